"""Layer norm, dropout and the classifier cost without a logits matrix, against plain float64 implementations.

Tolerances: u = 2^-24 is the largest relative rounding error of one fp32 operation.  A sum of k products of relative errors at most
u each, in any order, is off by at most k u sum|terms| and, with errors of either sign, by LAMBDA sqrt(k) u sum|terms| but for a
negligible share of inputs (Higham and Mary, "A new approach to probabilistic rounding error analysis", 2019; LAMBDA = 8)."""
import ctypes as C
import os

import numpy as np
import pytest

from kutil import call, capi, dev, dev_double, ws_bytes

U = 2.0 ** -24
LAMBDA = 8
EPS = 1e-5
TAIL = 64  # floats behind every output that no kernel may touch
MARK = np.float32(1234.5)


class Out(capi.DeviceBuffer):
    """An output of `shape` filled with NaN (write-only outputs must not read it), or with `start`, with marks behind it."""

    def __init__(self, shape, start=None):
        self.want, self.count = shape, int(np.prod(shape))
        a = np.full(self.count + TAIL, MARK, np.float32)
        a[:self.count] = np.nan if start is None else np.asarray(start, np.float32).ravel()
        super().__init__(array=a)

    def get(self):
        a = self.numpy()
        assert np.all(a[self.count:] == MARK), 'wrote behind the end'
        return a[:self.count].reshape(self.want).copy()


def within(got, want, bound, what):
    got = got.astype(np.float64)
    bound = np.broadcast_to(bound, want.shape)
    assert np.array_equal(np.isfinite(got), np.isfinite(want)), what
    f = np.isfinite(want)
    err = np.abs(got[f] - want[f])
    bad = err > bound[f]
    assert not bad.any(), '%s: %d of %d off, worst %.3g over a bound of %.3g' % (
        what, bad.sum(), bad.size, err[bad].max(), bound[f][bad][np.argmax(err[bad])])


def sum_err(k):
    return min(k, LAMBDA * np.sqrt(k)) * U


def need(name, *a):
    """A workspace full of NaNs: nothing may be read from it that was not written."""
    b = ws_bytes(name, *a)
    return capi.DeviceBuffer(array=np.full(max(b, 16), 0xFF, np.uint8)), b


# ------------------------------------------------------------------------------------------------------------- layer norm
def norm_ref(x, gain, bias):
    mean = x.mean(0)
    var = ((x - mean) ** 2).mean(0)
    r = 1 / np.sqrt(var + EPS)
    return gain[:, None] * ((x - mean) * r) + bias[:, None], mean, r


def norm_bounds(x, gain, bias, mean, r):
    """Error of the mean, relative error of r, error of y."""
    f = x.shape[0]
    amax = np.abs(x).max(0)
    e_mean = sum_err(f) * np.abs(x).mean(0) + 4 * U * amax
    # var: deviations off by e_mean and 2u each, squares summed; r has half of var's relative error
    dev_rms = np.sqrt(((x - mean) ** 2).mean(0))
    e_r = 0.5 * (sum_err(f) + 8 * U + (2 * e_mean * dev_rms + e_mean ** 2 + 2 * U * amax * dev_rms) * r ** 2) + 4 * U
    xh = np.abs((x - mean) * r)
    e_xh = (e_mean + 2 * U * amax) * r + xh * (e_r + 4 * U)
    return e_mean, e_r, np.abs(gain)[:, None] * (e_xh + 2 * U * xh) + 2 * U * (np.abs(gain[:, None]) * xh + np.abs(bias)[:, None]), e_xh


def norm_data(f, n, seed, offset=2.0):
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((f, n)) * (0.5 + 2 * rng.random(n)) + rng.standard_normal(n) * offset).astype(np.float32)
    gain = (1 + 0.2 * rng.standard_normal(f)).astype(np.float32)
    bias = (0.2 * rng.standard_normal(f)).astype(np.float32)
    return x, gain, bias, rng.standard_normal((f, n)).astype(np.float32)


NORM_SHAPES = [(1, 1), (1, 5), (2, 1), (3, 64), (5, 3), (16, 16), (63, 65), (64, 4), (160, 128), (160, 37), (257, 12), (512, 1),
               (512, 128), (1000, 31), (1025, 8), (2048, 20), (2049, 64), (4096, 36), (4097, 16), (9075, 5), (9075, 128), (40000, 1),
               (20000, 4), (33, 5000), (128, 3010), (7, 20001),
               (512, 8260), (513, 8263), (4100, 1030), (30000, 20), (30001, 100), (70000, 3)]


@pytest.mark.gpu
@pytest.mark.parametrize('f,n', NORM_SHAPES)
def test_layer_norm(f, n):
    x, gain, bias, _ = norm_data(f, n, f * 131 + n)
    want, mean, r = norm_ref(x.astype(np.float64), gain.astype(np.float64), bias.astype(np.float64))
    e_mean, e_r, e_y, _ = norm_bounds(x.astype(np.float64), gain, bias, mean, r)
    y, st = Out((f, n)), Out((2, n))
    ws, size = need('mcn_layer_norm_workspace_bytes', f, n)
    dx, dg, db = dev(x), dev(gain), dev(bias)
    call('mcn_layer_norm', dx, dg, db, y, st, f, n, EPS, ws, size, None)
    got, stats = y.get(), st.get()
    within(stats[0], mean, e_mean, 'mean')
    within(stats[1], r, e_r * r, 'r')
    within(got, want, e_y, 'y')
    # without gains, biases and statistics, in place, and at an address that is not 16-byte aligned
    z = Out((f * n + 1,), np.concatenate([[0], x.ravel()]))
    call('mcn_layer_norm', z.ptr + 4, None, None, z.ptr + 4, None, f, n, EPS, ws, size, None)
    one, zero = np.ones(f), np.zeros(f)
    want1, _, _ = norm_ref(x.astype(np.float64), one, zero)
    within(z.get()[1:].reshape(f, n), want1, norm_bounds(x.astype(np.float64), one, zero, mean, r)[2], 'y in place')


@pytest.mark.gpu
@pytest.mark.parametrize('offset', [1e3, 1e5])
def test_layer_norm_far_from_zero(offset):
    """Large means: a variance formed as a difference of two large sums would lose everything."""
    x, gain, bias, _ = norm_data(700, 24, 5, offset)
    x64 = x.astype(np.float64)
    want, mean, r = norm_ref(x64, gain.astype(np.float64), bias.astype(np.float64))
    y, st = Out((700, 24)), Out((2, 24))
    ws, size = need('mcn_layer_norm_workspace_bytes', 700, 24)
    keep = dev(x), dev(gain), dev(bias)
    call('mcn_layer_norm', *keep, y, st, 700, 24, EPS, ws, size, None)
    within(y.get(), want, norm_bounds(x64, gain, bias, mean, r)[2], 'y')


@pytest.mark.gpu
def test_layer_norm_one_bad_case_stays_alone():
    """An infinity or NaN in one case changes that case only; a constant case gives the biases."""
    x, gain, bias, _ = norm_data(300, 40, 9)
    x[7, 3], x[8, 11], x[:, 20] = np.inf, np.nan, 3.25
    y = Out((300, 40))
    ws, size = need('mcn_layer_norm_workspace_bytes', 300, 40)
    keep = dev(x), dev(gain), dev(bias)
    call('mcn_layer_norm', *keep, y, None, 300, 40, EPS, ws, size, None)
    got = y.get()
    assert not np.isfinite(got[:, 11]).any() and not np.isfinite(got[7, 3])
    fine = [c for c in range(40) if c not in (3, 11)]
    want, mean, r = norm_ref(x[:, fine].astype(np.float64), gain.astype(np.float64), bias.astype(np.float64))
    within(got[:, fine], want, norm_bounds(x[:, fine].astype(np.float64), gain, bias, mean, r)[2], 'the other cases')


def undo_ref(g, x, gain, mean, r):
    h, xh = gain[:, None] * g, (x - mean) * r
    return r * (h - h.mean(0) - xh * (h * xh).mean(0)), (g * xh).sum(1), g.sum(1)


def undo_bounds(g, x, gain, bias, mean, r):
    f, n = x.shape
    _, e_r, _, e_xh = norm_bounds(x, gain, bias, mean, r)
    h, xh = gain[:, None] * g, (x - mean) * r
    e_m1 = (sum_err(f) + 4 * U) * np.abs(h).mean(0)
    e_m2 = (sum_err(f) + 6 * U) * np.abs(h * xh).mean(0) + (np.abs(h) * e_xh).mean(0)
    m2 = np.abs((h * xh).mean(0))
    mag = np.abs(h) + np.abs(h.mean(0)) + np.abs(xh) * m2
    e_dx = r * (e_m1 + np.abs(xh) * e_m2 + e_xh * m2 + 6 * U * mag + e_r * mag)
    e_dg = (sum_err(n) + 4 * U) * np.abs(g * xh).sum(1) + (np.abs(g) * e_xh).sum(1)
    return e_dx, e_dg, (sum_err(n) + 2 * U) * np.abs(g).sum(1)


@pytest.mark.gpu
@pytest.mark.parametrize('f,n', NORM_SHAPES)
def test_layer_norm_undo(f, n):
    x, gain, bias, g = norm_data(f, n, f * 17 + n)
    X, G, g64 = x.astype(np.float64), gain.astype(np.float64), g.astype(np.float64)
    _, mean, r = norm_ref(X, G, bias.astype(np.float64))
    wx, wg, wb = undo_ref(g64, X, G, mean, r)
    ex, eg, eb = undo_bounds(g64, X, G, bias, mean, r)
    st = Out((2, n), np.stack([mean, r]))
    dx, dg, db = Out((f, n)), Out((f,)), Out((f,))
    ws, size = need('mcn_layer_norm_undo_workspace_bytes', f, n)
    kg, kx, ka = dev(g), dev(x), dev(gain)
    call('mcn_layer_norm_undo', kg, kx, ka, st, dx, dg, db, f, n, 0.0, 1.0, 0.0, 1.0, 0.0, 1.0, ws, size, None)
    first = dx.get(), dg.get(), db.get()
    within(first[0], wx, ex, 'dx')
    within(first[1], wg, eg, 'dgain')
    within(first[2], wb, eb, 'dbias')
    # again: the same bits
    call('mcn_layer_norm_undo', kg, kx, ka, st, dx, dg, db, f, n, 0.0, 1.0, 0.0, 1.0, 0.0, 1.0, ws, size, None)
    for a, b in zip(first, (dx.get(), dg.get(), db.get())):
        assert np.array_equal(a, b)
    # added onto what is there, scaled; then each output alone
    t, tg, tb = (np.random.default_rng(1).standard_normal(s).astype(np.float32) for s in ((f, n), (f,), (f,)))
    dx, dg, db = Out((f, n), t), Out((f,), tg), Out((f,), tb)
    call('mcn_layer_norm_undo', kg, kx, ka, st, dx, dg, db, f, n, 1.0, 0.5, 0.9, -0.25, 0.5, 2.0, ws, size, None)
    within(dx.get(), t + 0.5 * wx, 0.5 * ex + 4 * U * (np.abs(t) + np.abs(wx)), 'dx added')
    within(dg.get(), 0.9 * tg - 0.25 * wg, 0.25 * eg + 4 * U * (np.abs(tg) + np.abs(wg)), 'dgain added')
    within(db.get(), 0.5 * tb + 2 * wb, 2 * eb + 4 * U * (np.abs(tb) + 2 * np.abs(wb)), 'dbias added')
    for k in range(3):
        outs = [Out((f, n)), Out((f,)), Out((f,))]
        args = [o if i == k else None for i, o in enumerate(outs)]
        call('mcn_layer_norm_undo', kg, kx, ka, st, *args, f, n, 0.0, 1.0, 0.0, 1.0, 0.0, 1.0, ws, size, None)
        assert np.array_equal(outs[k].get(), first[k])
    # no gains; operands that are not 16-byte aligned
    ug, ux = dev(np.concatenate([[0], g.ravel()])), dev(np.concatenate([[0], x.ravel()]))
    dx = Out((f * n + 1,))
    call('mcn_layer_norm_undo', ug.ptr + 4, ux.ptr + 4, None, st, dx.ptr + 4, None, None, f, n, 0.0, 1.0, 0.0, 1.0, 0.0, 1.0, ws, size, None)
    one = np.ones(f)
    within(dx.get()[1:].reshape(f, n), undo_ref(g64, X, one, mean, r)[0], undo_bounds(g64, X, one, bias, mean, r)[0], 'dx, no gains')


@pytest.mark.gpu
@pytest.mark.parametrize('f,n', [(24, 7), (130, 16)])
def test_layer_norm_undo_against_differences(f, n):
    """d sum(g y) along random directions, central differences of the float64 formula.

    Differences: step 1e-4, error O(step^2) times third derivatives of order one: 1e-6 of the sum of magnitudes is ample."""
    x, gain, bias, g = norm_data(f, n, 3)
    X, G, B = (a.astype(np.float64) for a in (x, gain, bias))
    _, mean, r = norm_ref(X, G, B)
    outs = Out((f, n)), Out((f,)), Out((f,))
    st = Out((2, n), np.stack([mean, r]))
    ws, size = need('mcn_layer_norm_undo_workspace_bytes', f, n)
    keep = dev(g), dev(x), dev(gain)
    call('mcn_layer_norm_undo', *keep, st, *outs, f, n, 0.0, 1.0, 0.0, 1.0, 0.0, 1.0, ws, size, None)
    got = [o.get().astype(np.float64) for o in outs]
    bounds = undo_bounds(g.astype(np.float64), X, G, B, mean, r)
    rng = np.random.default_rng(4)
    for k in range(3):
        d = [np.zeros_like(X), np.zeros_like(G), np.zeros_like(B)]
        d[k] = rng.standard_normal(d[k].shape)
        h = 1e-4
        value = lambda s: (g * norm_ref(X + s * d[0], G + s * d[1], B + s * d[2])[0]).sum()  # noqa: E731
        want = (value(h) - value(-h)) / (2 * h)
        assert abs((got[k] * d[k]).sum() - want) <= (bounds[k] * np.abs(d[k])).sum() + 1e-6 * (np.abs(got[k] * d[k])).sum()


@pytest.mark.gpu
@pytest.mark.parametrize('f,n', [(2, 1 << 20), (16, 1 << 18)])
def test_layer_norm_undo_sums_long_rows_in_short_chains(f, n):
    """Equal terms, whose rounding errors all go the same way: the error of a row's sum is the number of additions one after the other
    times u.  n / 1024 by a thread, 2 over the lanes of a row, 64 + 16 over the blocks' partial sums, and 2 u for the product and the output:
    at most 340 u (one wave along the whole row would add n / 64 terms: 2590 u and 646 u for 0.1)."""
    x = np.where(np.arange(f) % 2 == 0, 1, -1).astype(np.float32)[:, None] * np.ones((1, n), np.float32)
    g = np.full((f, n), 0.1, np.float32)
    r = np.float32(1 / np.sqrt(1 + EPS))
    st = Out((2, n), np.stack([np.zeros(n), np.full(n, r)]))
    dg, db = Out((f,)), Out((f,))
    ws, size = need('mcn_layer_norm_undo_workspace_bytes', f, n)
    keep = dev(g), dev(x), dev(np.ones(f, np.float32))
    call('mcn_layer_norm_undo', *keep, st, None, dg, db, f, n, 0.0, 1.0, 0.0, 1.0, 0.0, 1.0, ws, size, None)
    term = n * float(np.float32(0.1))
    within(db.get(), np.full(f, term), 340 * U * term, 'dbias')
    within(dg.get(), term * float(r) * x[:, 0].astype(np.float64), 340 * U * term, 'dgain')


@pytest.mark.gpu
@pytest.mark.parametrize('n', [1, 4, 7, 3755])
def test_layer_norm_of_two_features_rounds_like_the_formula(n):
    """With two features h - mean(h) - xh mean(h xh) cancels down to rounding errors: the same ones as of the formula in float32, one
    operation after the other (two terms have one order), so the same bits."""
    f = np.float32
    rng = np.random.default_rng(9)
    x, g = rng.standard_normal((2, n)).astype(f) * 2 + 1, rng.standard_normal((2, n)).astype(f)
    gain, bias = (1 + 0.2 * rng.standard_normal(2)).astype(f), rng.standard_normal(2).astype(f)
    mean = (x[0] + x[1]) / f(2)
    d = x - mean
    r = f(1) / np.sqrt((d[0] * d[0] + d[1] * d[1]) / f(2) + f(EPS))
    xh = d * r
    h = gain[:, None] * g
    m1, m2 = (h[0] + h[1]) / f(2), (h[0] * xh[0] + h[1] * xh[1]) / f(2)
    y, st, dx = Out((2, n)), Out((2, n)), Out((2, n))
    ws, size = need('mcn_layer_norm_workspace_bytes', 2, n)
    wu, sizeu = need('mcn_layer_norm_undo_workspace_bytes', 2, n)
    kx, kg, kgain, kbias = dev(x), dev(g), dev(gain), dev(bias)
    call('mcn_layer_norm', kx, kgain, kbias, y, st, 2, n, EPS, ws, size, None)
    call('mcn_layer_norm_undo', kg, kx, kgain, st, dx, None, None, 2, n, 0.0, 1.0, 0.0, 1.0, 0.0, 1.0, wu, sizeu, None)
    assert np.array_equal(st.get(), np.stack([mean, r]))
    assert np.array_equal(y.get(), gain[:, None] * xh + bias[:, None])
    assert np.array_equal(dx.get(), r * ((h - m1) - xh * m2))


# ------------------------------------------------------------------------------------------------------------- dropout
def philox_words(count, seed, step, first_quad=0):
    """Philox-4x32, ten rounds, in Python integers' width by uint64 arithmetic."""
    low, quads = np.uint64(0xFFFFFFFF), (count + 3) // 4
    q = np.arange(quads, dtype=np.uint64) + np.uint64(first_quad)
    c = [q & low, q >> np.uint64(32), np.full_like(q, step & 0xFFFFFFFF), np.full_like(q, step >> 32)]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, 1).astype(np.uint32).ravel()[:count]


def kept(count, p, seed, step):
    return philox_words(count, seed, step).astype(np.uint64) >= np.uint64(int(float(np.float32(p)) * 2.0 ** 32))


@pytest.mark.gpu
@pytest.mark.parametrize('n', [1, 3, 4, 5, 1023, 20480, 4213 * 37, 1 << 20])
@pytest.mark.parametrize('p', [0.0, 0.4, 0.999])
def test_dropout(n, p):
    rng = np.random.default_rng(n)
    x = rng.standard_normal(n).astype(np.float32)
    seed, step = (0xDEADBEEF << 32) + n, (5 << 32) + 17
    keep = kept(n, p, seed, step)
    scale = 1 / (1 - float(np.float32(p)))
    want = np.where(keep, x * scale, 0.0)
    y, dx = Out((n,)), dev(x)
    call('mcn_dropout', dx, y, n, p, seed, step, None, 0.0, 1.0, None)
    got = y.get()
    assert np.array_equal(got != 0, keep & (x != 0))
    within(got, want, 2 * U * np.abs(want), 'y')
    # in place, and at an address that is not 16-byte aligned: the same bits
    z = Out((n + 1,), np.concatenate([[0], x]))
    call('mcn_dropout', z.ptr + 4, z.ptr + 4, n, p, seed, step, None, 0.0, 1.0, None)
    assert np.array_equal(z.get()[1:], got)
    # added onto what is there; step given in parts, one of them in device memory
    t = rng.standard_normal(n).astype(np.float32)
    y = Out((n,), t)
    counter = capi.DeviceBuffer(array=np.array([step - 20], np.uint64))
    call('mcn_counter_add', counter.ptr, 9, None)
    call('mcn_dropout', dx, y, n, p, seed, 11, counter.ptr, 0.5, -2.0, None)
    within(y.get(), 0.5 * t - 2 * want, 4 * U * (np.abs(t) + 2 * np.abs(want)), 'added')


@pytest.mark.gpu
def test_dropout_masked_places_do_not_come_through():
    n, p = 4096, 0.5
    keep = kept(n, p, 7, 9)
    x = np.where(keep, 1.0, np.nan).astype(np.float32)
    x[~keep & (np.arange(n) % 3 == 0)] = np.inf
    y, dx = Out((n,)), dev(x)
    call('mcn_dropout', dx, y, n, p, 7, 9, None, 0.0, 1.0, None)
    assert np.array_equal(y.get(), np.where(keep, np.float32(2), np.float32(0)))


@pytest.mark.gpu
def test_dropout_statistics():
    """Share kept: 2^20 draws of probability 0.6 have a standard deviation of 5e-4 of the share; five of them are allowed.  Masks of
    neighbouring steps and seeds agree on a share of 0.6^2 + 0.4^2 = 0.52, likewise."""
    n = 1 << 20
    one = dev(np.ones(n, np.float32))
    masks = []
    for seed, step in ((1, 1), (1, 2), (2, 1)):
        y = Out((n,))
        call('mcn_dropout', one, y, n, 0.4, seed, step, None, 0.0, 1.0, None)
        masks.append(y.get() != 0)
        assert abs(masks[-1].mean() - 0.6) < 2.5e-3
    for a, b in ((0, 1), (0, 2), (1, 2)):
        assert abs((masks[a] == masks[b]).mean() - 0.52) < 2.5e-3


# ------------------------------------------------------------------------------------------------------------- classifier cost
def fcl_data(d, v, n, seed, masked=0.0, padded=0, lean=6.0, least=0.0):
    rng = np.random.default_rng(seed)
    w = (rng.standard_normal((v, d)) / np.sqrt(d)).astype(np.float32)
    labels = rng.integers(v, size=n)
    x = (rng.standard_normal((d, n)) + (least + lean * rng.random(n)) * w[labels].T).astype(np.float32)
    b = (0.1 * rng.standard_normal(v)).astype(np.float32)
    if masked:
        hide = rng.random(v) < masked
        hide[labels] = False
        b[hide] = -np.inf
    lab = labels.astype(np.float32)
    if padded:
        lab[n - padded:] = -1
    return w, x, b, lab


def fcl_ref(w, x, b, lab, coeff):
    w, x, b = (a.astype(np.float64) for a in (w, x, b))
    v, n = w.shape[0], x.shape[1]
    z = w @ x + b[:, None]
    top = z.max(0)
    e = np.exp(z - top)
    tot = e.sum(0)
    ok = (lab >= 0) & (lab < v)
    li = np.where(ok, lab, 0).astype(int)
    at = z[li, np.arange(n)]
    logp = np.where(ok, at - top - np.log(tot), 0.0)
    correct = np.where(ok & (at == top), 1.0 / (z == top).sum(0), 0.0)
    dz = -e / tot
    dz[li, np.arange(n)] += 1
    dz *= coeff * ok
    # the error of one logit, per case; of e / tot, relative; of dz
    a = np.abs(w) @ np.abs(x) + np.where(np.isfinite(b), np.abs(b), 0)[:, None]
    ez = (sum_err(w.shape[1]) + 4 * U) * a.max(0)
    er = 2 * ez + sum_err(v) + 16 * U
    # p is off by p (sum over the others of p times twice the error of a logit) -- the error of its own logit cancels, the two calls'
    # logits being the same -- and by the rounding of the sum: of what is not at the maximum, and of the whole
    p = e / tot
    edz = (np.abs(coeff) * ok) * p * ((1 - p) * 2 * ez + sum_err(v) * (1 - p.max(0)) + 16 * U) + 4 * U * np.abs(dz)
    return dict(z=z, top=top, tot=tot, logp=logp, correct=correct, dz=dz, dx=w.T @ dz, dw=dz @ x.T, db=dz.sum(1), ez=ez, er=er, ok=ok,
                edx=np.abs(w).T @ edz + (sum_err(v) + 2 * U) * (np.abs(w).T @ np.abs(dz)),
                edw=edz @ np.abs(x).T + (sum_err(n) + 2 * U) * (np.abs(dz) @ np.abs(x).T),
                edb=edz.sum(1) + (sum_err(n) + 2 * U) * np.abs(dz).sum(1))


def check_forward(ref, stats, logp, correct, what=''):
    within(stats[0], ref['top'], ref['ez'] + 2 * U * np.abs(ref['top']), what + 'max')
    within(stats[1], ref['tot'], ref['tot'] * ref['er'], what + 'sum')
    within(logp, ref['logp'], 2 * ref['er'] + 4 * U * np.abs(ref['logp']), what + 'logp')
    # decisions: where the two largest logits are further apart than their errors
    z = np.sort(ref['z'], 0)
    clear = z[-1] - z[-2] > 4 * ref['ez'] if z.shape[0] > 1 else np.ones(z.shape[1], bool)
    assert np.array_equal(correct[clear], ref['correct'][clear].astype(np.float32)), what + 'correct'


# inputs, outputs, cases
FCL_SHAPES = [(1, 1, 1), (1, 2, 3), (3, 1, 5), (16, 2, 1), (160, 4213, 1), (160, 4213, 2), (33, 65, 7), (64, 64, 64), (32, 128, 128),
              (160, 1000, 128), (512, 1999, 128), (100, 333, 129), (17, 4097, 33), (513, 130, 260), (1000, 257, 31), (2049, 96, 40),
              (128, 640, 512), (96, 10575, 100), (256, 300, 1025), (48, 20000, 17), (200, 70, 48), (96, 600, 63), (96, 600, 64),
              (96, 600, 65), (1031, 8200, 20), (2050, 4200, 3), (40, 4400, 100),
              (300, 5600, 130), (20, 70000, 70)]


def fcl_run(w, x, b, lab, coeff=1.0, scales=(0.0, 0.0, 1.0, 0.0, 1.0), start=(None, None, None), stream=None):
    (v, d), n = w.shape, x.shape[1]
    st, lp, ok = Out((2, n)), Out((n,)), Out((n,))
    dx, dw, db = Out((d, n), start[0]), Out((v, d), start[1]), Out((v,), start[2])
    cost = dev_double(2)
    ws, size = need('mcn_fc_logreg_workspace_bytes', d, v, n, 1)
    keep = dev(w), dev(x), dev(b) if b is not None else None, dev(lab)
    call('mcn_fc_logreg_cost', *keep, st, lp, ok, d, v, n, cost, ws, size, stream)
    call('mcn_fc_logreg_grad', *keep, st, dx, dw, db, d, v, n, coeff, *scales, ws, size, stream)
    return [o.get() for o in (st, lp, ok, dx, dw, db)] + [cost.numpy()]


@pytest.mark.gpu
@pytest.mark.parametrize('d,v,n', FCL_SHAPES)
def test_fc_logreg(d, v, n):
    w, x, b, lab = fcl_data(d, v, n, d * 7 + v + n, masked=0.1 if v > 50 else 0, padded=n // 4)
    coeff = 0.37
    ref = fcl_ref(w, x, b, lab, coeff)
    st, lp, ok, dx, dw, db, cost = first = fcl_run(w, x, b, lab, coeff)
    check_forward(ref, st, lp, ok)
    within(dx, ref['dx'], ref['edx'], 'dx')
    within(dw, ref['dw'], ref['edw'], 'dw')
    within(db, ref['db'], ref['edb'], 'db')
    assert abs(cost[0] + lp.astype(np.float64).sum()) <= 1e-12 * n + 1e-12 * np.abs(lp).sum()
    assert cost[1] == pytest.approx(ref['ok'].sum() - ok.astype(np.float64).sum(), abs=1e-9)
    for a, c in zip(first, fcl_run(w, x, b, lab, coeff)):
        assert np.array_equal(a, c), 'not the same bits again'
    # added onto what is there, with scales; no biases
    rng = np.random.default_rng(2)
    t = [rng.standard_normal(s).astype(np.float32) for s in ((d, n), (v, d), (v,))]
    ref = fcl_ref(w, x, np.zeros(v), lab, coeff)
    got = fcl_run(w, x, None, lab, coeff, (1.0, 0.9, 0.5, 0.25, -2.0), t)
    within(got[3], t[0] + ref['dx'], ref['edx'] + 4 * U * (np.abs(t[0]) + np.abs(ref['dx'])), 'dx added')
    within(got[4], 0.9 * t[1] + 0.5 * ref['dw'], 0.5 * ref['edw'] + 4 * U * (np.abs(t[1]) + np.abs(ref['dw'])), 'dw added')
    within(got[5], 0.25 * t[2] - 2 * ref['db'], 2 * ref['edb'] + 4 * U * (np.abs(t[2]) + 2 * np.abs(ref['db'])), 'db added')


def fcl_forms(d, v, n, backward):
    """(classes, tiles of the logits, k blocks of a share of the input gradient, shares, gradients' tiles two to a CU) of every piece."""
    lib = C.CDLL(os.path.join(os.path.dirname(capi.LIB_PATH), 'libmiconvnet_hooks.so'))  # (the test build: the same rules)
    out = (C.c_int * 50)()
    return [tuple(out[5 * i:5 * i + 5]) for i in range(lib.mcn_fc_logreg_test_forms(d, v, n, backward, out, 10))]


SHARED, WHOLE, HALF, FEW = range(4)


@pytest.mark.gpu
@pytest.mark.parametrize('d,v,n,logits,steps,shared', [
    (160, 10575, 509, SHARED, 9, True),
    (96, 10575, 509, SHARED, 9, False),   # two tiles a CU, several tiles of cases, the last of them in part
    (300, 70000, 70, WHOLE, 9, True),     # more steps of 32 features than there are stages
    (1000, 15000, 1025, WHOLE, 64, True),  # shares of more classes than exponents are loaded at a time, of groups of different scales
    (600, 33000, 260, SHARED, 9, True),
    (512, 10575, 128, HALF, 9, True),
    (100, 333, 129, HALF, 1, False),
    (96, 600, 64, FEW, 1, False)])
def test_fc_logreg_every_form_on_dense_operands(d, v, n, logits, steps, shared):
    for backward in (0, 1):
        forms = fcl_forms(d, v, n, backward)
        assert len(forms) == 1 and forms[0][1] == logits and forms[0][2] >= steps and (not backward or forms[0][4] == shared), forms
    w, x, b, lab = fcl_data(d, v, n, 43, masked=0.05, padded=n // 10)
    rng = np.random.default_rng(44)
    w *= np.repeat(np.float32(10.0) ** rng.choice([-7, -3, 0], (v + 31) // 32), 32)[:v, None]  # (32 classes have one scale)
    ref = fcl_ref(w, x, b, lab, 0.37)
    st, lp, ok, dx, dw, db, cost = fcl_run(w, x, b, lab, 0.37)
    check_forward(ref, st, lp, ok)
    for got, k in ((dx, 'dx'), (dw, 'dw'), (db, 'db')):
        within(got, ref[k], ref['e' + k], k)


@pytest.mark.gpu
@pytest.mark.parametrize('d,v,n', [(20000, 5000, 70), (20000, 5600, 8)])
def test_fc_logreg_of_more_classes_than_a_piece_takes(d, v, n):
    """Two pieces, the last one with a short rest; three, the last one short."""
    rng = np.random.default_rng(71)
    w = rng.standard_normal((v, d), dtype=np.float32) * np.float32(d ** -0.5)
    x = rng.standard_normal((d, n), dtype=np.float32)
    b = (0.1 * rng.standard_normal(v)).astype(np.float32)
    lab = rng.integers(v, size=n).astype(np.float32)
    lab[:4] = 0, 2431, 2432, v - 1
    ref = fcl_ref(w, x, b, lab, 0.5)
    st, lp, ok, dx, dw, db, cost = fcl_run(w, x, b, lab, 0.5)
    check_forward(ref, st, lp, ok)
    for got, k in ((dx, 'dx'), (dw, 'dw'), (db, 'db')):
        within(got, ref[k], ref['e' + k], k)


@pytest.mark.gpu
@pytest.mark.parametrize('d,v,n', [(580, 23, 52), (512, 5, 3), (160, 4213, 64), (160, 4213, 65), (512, 1000, 128), (96, 33000, 20), (2000, 5000, 16)])
def test_fc_logreg_of_certain_cases(d, v, n):
    """Labels whose probability is 1 - 1e-3 to 1 - 1e-8: the gradient is what is left of 1 - p."""
    w, x, b, lab = fcl_data(d, v, n, 61, lean=10.0, least=14.0)
    ref = fcl_ref(w, x, b, lab, 1.0)
    st, lp, ok, dx, dw, db, cost = fcl_run(w, x, b, lab)
    check_forward(ref, st, lp, ok)
    for got, k in ((dx, 'dx'), (dw, 'dw'), (db, 'db')):
        within(got, ref[k], ref['e' + k], k)


@pytest.mark.gpu
@pytest.mark.parametrize('d,v,n', [(33, 65, 7), (160, 1000, 128), (100, 700, 300)])
def test_fc_logreg_each_gradient_alone_and_unaligned(d, v, n):
    w, x, b, lab = fcl_data(d, v, n, 11)
    st, lp, ok, *grads, _ = fcl_run(w, x, b, lab, 0.5)
    ws, size = need('mcn_fc_logreg_workspace_bytes', d, v, n, 1)
    shift = lambda a: dev(np.concatenate([[0], a.ravel()]))  # noqa: E731
    keep = [shift(a) for a in (w, x, b, lab)]
    ptrs = [k.ptr + 4 for k in keep]
    st2, lp2, ok2 = Out((2 * n + 1,)), Out((n + 1,)), Out((n + 1,))
    call('mcn_fc_logreg_cost', *ptrs, st2.ptr + 4, lp2.ptr + 4, ok2.ptr + 4, d, v, n, None, ws, size, None)
    ref = fcl_ref(w, x, b, lab, 0.5)
    check_forward(ref, st2.get()[1:].reshape(2, n), lp2.get()[1:], ok2.get()[1:], 'unaligned ')
    shapes = ((d, n), (v, d), (v,))
    for k in range(3):
        outs = [Out((int(np.prod(s)) + 1,)) for s in shapes]
        args = [o.ptr + 4 if i == k else None for i, o in enumerate(outs)]
        call('mcn_fc_logreg_grad', *ptrs, st2.ptr + 4, *args, d, v, n, 0.5, 0.0, 0.0, 1.0, 0.0, 1.0, ws, size, None)
        name = ('dx', 'dw', 'db')[k]
        within(outs[k].get()[1:].reshape(shapes[k]), ref[name], ref['e' + name], 'unaligned ' + name)


@pytest.mark.gpu
@pytest.mark.parametrize('n', [1, 6, 140])
def test_fc_logreg_ties_and_masks(n):
    """Equal classes tie exactly wherever they stand; masked classes, cases without a label, cases with no class left."""
    d, v = 20, 400
    w, x, b, lab = fcl_data(d, v, n, 13, lean=0)
    lab[:] = 7
    dirs = x / np.linalg.norm(x, axis=0)
    if n == 1:
        w[[7, 70, 250, 399]] = dirs[:, 0]  # far ahead of the others, and the same
        w[[7, 70, 250, 399]] *= 100
        b[[7, 70, 250, 399]] = 0.5
        st, lp, ok, dx, dw, db, cost = fcl_run(w, x, b, lab)
        assert ok[0] == 0.25 and cost[1] == 0.75
        assert np.array_equal(dw[70], dw[250]) and db[7] == pytest.approx(0.75, rel=1e-5)
        return
    # the lowest value of the type, and minus infinity, as masks
    for low in (-np.inf, np.finfo(np.float32).min):
        b2 = b.copy()
        b2[50:390] = low
        st, lp, ok, dx, dw, db, _ = fcl_run(w, x, b2, lab)
        ref = fcl_ref(w, x, b2, lab, 1.0)
        check_forward(ref, st, lp, ok, 'masked ') if low == -np.inf else within(lp, ref['logp'], 2 * ref['er'] + 4 * U * np.abs(ref['logp']) + 1e-5, 'logp')
        assert not dw[50:390].any() and not db[50:390].any()
    # no class left
    st, lp, ok, dx, dw, db, _ = fcl_run(w, x, np.full(v, -np.inf, np.float32), lab)
    assert np.all(st[0] == -np.inf) and not st[1].any() and np.all(lp == -np.inf) and not ok.any()
    assert not dx.any() and not dw.any() and not db.any()
    # no labels: out of range on either side, not a number
    for bad in (-1, v, 1e9, np.nan, np.inf, -np.inf):
        st, lp, ok, dx, dw, db, cost = fcl_run(w, x, b, np.full(n, bad, np.float32))
        assert not lp.any() and not ok.any() and not cost.any() and not dx.any() and not dw.any() and not db.any()


@pytest.mark.gpu
@pytest.mark.parametrize('bad', [np.nan, np.inf, 1e38])
@pytest.mark.parametrize('n', [1, 6, 40, 140])
def test_fc_logreg_masked_places_do_not_come_through(n, bad):
    """Weights of classes that are taken out and inputs of cases that do not count: whatever they hold."""
    d, v = 36, 500
    w, x, b, lab = fcl_data(d, v, n, 31, masked=0.2, padded=n // 3)
    out, off = np.isneginf(b), lab < 0
    assert out.any()
    w0, x0 = w.copy(), x.copy()
    w0[out], x0[:, off] = 0, 0
    w[out], x[:, off] = bad, bad
    ref = fcl_ref(w0, x0, b, lab, 0.5)
    st, lp, ok, dx, dw, db, _ = fcl_run(w, x, b, lab, 0.5)
    keep = ~off
    within(st[:, keep], np.stack([ref['top'], ref['tot']])[:, keep], np.stack([ref['ez'] + 2 * U * np.abs(ref['top']), ref['tot'] * ref['er']])[:, keep], 'stats')
    within(lp, ref['logp'], 2 * ref['er'] + 4 * U * np.abs(ref['logp']), 'logp')
    for got, k in ((dx, 'dx'), (dw, 'dw'), (db, 'db')):
        within(got, ref[k], ref['e' + k], k)
    assert not dx[:, off].any() and not dw[out].any()


@pytest.mark.gpu
@pytest.mark.parametrize('bad', [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize('n', [6, 140])
def test_fc_logreg_cases_that_do_not_count_have_no_gradient_whatever_the_weights_hold(n, bad):
    """A class that takes part has a weight that is no number: the padded cases' input gradients are zero all the same, and added as such."""
    d, v = 36, 500
    w, x, b, lab = fcl_data(d, v, n, 34, padded=n // 3)
    off = lab < 0
    w[77, 5] = bad
    assert not fcl_run(w, x, b, lab, 0.5)[3][:, off].any()
    t = np.random.default_rng(3).standard_normal((d, n)).astype(np.float32)
    assert np.array_equal(fcl_run(w, x, b, lab, 0.5, (0.5, 0.0, 1.0, 0.0, 1.0), (t, None, None))[3][:, off], np.float32(0.5) * t[:, off])


def fcl_check(ref, got, cases, feats):
    """Statistics and costs of `cases`, gradients of `feats`, against a reference."""
    st, lp, ok, dx, dw, db, _ = got
    within(st[:, cases], np.stack([ref['top'], ref['tot']])[:, cases], np.stack([ref['ez'] + 2 * U * np.abs(ref['top']), ref['tot'] * ref['er']])[:, cases], 'stats')
    within(lp[cases], ref['logp'][cases], (2 * ref['er'] + 4 * U * np.abs(ref['logp']))[cases], 'logp')
    within(dx[feats][:, cases], ref['dx'][feats][:, cases], ref['edx'][feats][:, cases], 'dx')
    within(dw, ref['dw'], ref['edw'], 'dw')
    within(db, ref['db'], ref['edb'], 'db')


@pytest.mark.gpu
@pytest.mark.parametrize('d,v,n', [(36, 500, 6), (36, 500, 64), (36, 500, 65), (36, 500, 140), (600, 300, 70), (40, 9000, 520)])
def test_fc_logreg_minus_infinite_logits_of_live_classes(d, v, n):
    """Weights of -inf against positive inputs: the class is out as one with a bias of -inf is, on either side of the number of cases
    that takes the other products; only its own features' input gradients are 0 * inf.  Its neighbours' small weights keep their bits."""
    w, x, b, lab = fcl_data(d, v, n, 35, padded=n // 4)
    x[3:6] = np.abs(x[3:6]) + 0.1
    out = np.array([50, 51, v - 1])
    w[52:60] *= 1e-6
    lab[np.isin(lab, out)] = 1
    w0, b0 = w.copy(), b.copy()
    w0[out], b0[out] = 0, -np.inf
    w[50, 3], w[51, 4:6], w[v - 1, 3:6] = -np.inf, -np.inf, -np.inf
    ref = fcl_ref(w0, x, b0, lab, 0.5)
    got = fcl_run(w, x, b, lab, 0.5)
    feats = np.array([k for k in range(d) if k not in (3, 4, 5)])
    fcl_check(ref, got, slice(None), feats)
    on = lab >= 0
    assert np.isnan(got[3][3:6][:, on]).all() and not got[3][:, ~on].any()
    assert not got[4][out].any() and not got[5][out].any()


@pytest.mark.gpu
@pytest.mark.parametrize('n', [6, 140])
def test_fc_logreg_infinities_that_leave_no_number(n):
    """A logit of +inf, and infinities of both signs in one logit: no finite cost, and only for the cases that have them."""
    d, v = 36, 500
    w, x, b, lab = fcl_data(d, v, n, 36)
    x[3:5] = np.abs(x[3:5]) + 0.1
    x[5, ::2], x[5, 1::2] = 1, -1
    for k, (at, val) in enumerate([((60, 3), np.inf), ((60, slice(3, 5)), [np.inf, -np.inf])]):
        w2 = w.copy()
        w2[at] = val
        st, lp, ok, *_ = fcl_run(w2, x, b, lab)
        assert np.isnan(lp).all() and np.isnan(st[1]).all()
    w2 = w.copy()
    w2[60, 5] = np.inf  # +inf for the even cases, -inf for the odd ones
    lab[lab == 60] = 61
    b0 = b.copy()
    b0[60] = -np.inf
    ref = fcl_ref(w, x, b0, lab, 1.0)
    st, lp, ok, dx, dw, db, _ = fcl_run(w2, x, b, lab)
    assert np.isnan(lp[::2]).all()
    within(lp[1::2], ref['logp'][1::2], (2 * ref['er'] + 4 * U * np.abs(ref['logp']))[1::2], 'logp')


@pytest.mark.gpu
@pytest.mark.parametrize('n', [6, 70, 300])
def test_fc_logreg_infinite_weights_far_apart(n):
    """Infinities of one sign, and of both, at features far from each other; a NaN behind an infinity."""
    d, v = 700, 300
    w, x, b, lab = fcl_data(d, v, n, 46)
    for k in (3, 500, 699):
        x[k] = np.abs(x[k]) + 0.1
    lab[np.isin(lab, (50, 60, 70))] = 1
    out, b0, w0 = [50], b.copy(), w.copy()
    b0[out], w0[out] = -np.inf, 0
    w[50, [3, 500, 699]] = -np.inf
    fcl_check(fcl_ref(w0, x, b0, lab, 0.5), fcl_run(w, x, b, lab, 0.5), slice(None), np.array([k for k in range(d) if k not in (3, 500, 699)]))
    for row, at, vals in ((60, [3, 699], [-np.inf, np.inf]), (60, [500, 699], [np.inf, -np.inf]), (70, [3, 500], [-np.inf, np.nan]), (70, [3, 500], [np.nan, -np.inf])):
        w2 = w.copy()
        w2[row, at] = vals
        st, lp, *_ = fcl_run(w2, x, b, lab)
        assert np.isnan(lp).all() and np.isnan(st[1]).all()


@pytest.mark.gpu
@pytest.mark.parametrize('n', [6, 140])
def test_fc_logreg_infinite_inputs(n):
    """An input of +inf against negative weights takes every class out: the case has statistics (-inf, 0) and no gradient, and the others
    do not see it.  One with classes taken out by their bias as well, whose weights count for nothing."""
    d, v = 36, 500
    w, x, b, lab = fcl_data(d, v, n, 37)
    w[:, 5] = -np.abs(w[:, 5]) - 0.01
    b[100:140] = -np.inf
    w[100:140, 5] = 1
    lab[(lab >= 100) & (lab < 140)] = 7
    bad = np.array([1, n - 1])
    x0, lab0 = x.copy(), lab.copy()
    x0[5, bad], lab0[bad] = 0, -1
    x[5, bad] = np.inf
    ref = fcl_ref(w, x0, b, lab0, 0.5)
    got = fcl_run(w, x, b, lab, 0.5)
    others = np.array([k for k in range(n) if k not in bad])
    fcl_check(ref, got, others, np.arange(d))
    st, lp, ok, dx, dw, db, cost = got
    assert np.all(st[0, bad] == -np.inf) and not st[1, bad].any() and np.all(lp[bad] == -np.inf) and not ok[bad].any()
    assert not dx[:, bad].any()


@pytest.mark.gpu
@pytest.mark.parametrize('n', [1, 6, 140])
def test_fc_logreg_label_of_a_masked_class(n):
    """log p = -inf, and the gradients of the formula: the label's one stays, and takes that class's weights with it."""
    d, v = 36, 500
    w, x, b, lab = fcl_data(d, v, n, 32)
    b[100:140] = -np.inf
    lab[::2] = 100 + np.arange(n)[::2] % 40
    with np.errstate(invalid='ignore'):
        ref = fcl_ref(w, x, b, lab, 0.5)
    st, lp, ok, dx, dw, db, cost = fcl_run(w, x, b, lab, 0.5)
    assert np.all(np.isneginf(lp[::2])) and not ok[::2].any() and np.isposinf(cost[0])
    check_forward(ref, st, lp, ok)
    for got, k in ((dx, 'dx'), (dw, 'dw'), (db, 'db')):
        within(got, ref[k], ref['e' + k], k)


@pytest.mark.gpu
@pytest.mark.parametrize('n', [6, 140])
@pytest.mark.parametrize('large,tiny', [(1e4, 1e-30), (1e6, 1e-20), (1.0, 1e-12)])
def test_fc_logreg_weights_of_very_different_sizes(n, large, tiny):
    """Groups of classes with large and tiny weights beside each other, in either order: every sum stays in range."""
    d, v = 40, 400
    w, x, b, lab = fcl_data(d, v, n, 33, lean=0)
    w[:100] *= tiny
    w[100:200] *= large
    w[200:300] *= tiny
    x /= large
    ref = fcl_ref(w, x, b, lab, 0.5)
    st, lp, ok, dx, dw, db, _ = fcl_run(w, x, b, lab, 0.5)
    check_forward(ref, st, lp, ok)
    for got, k in ((dx, 'dx'), (dw, 'dw'), (db, 'db')):
        within(got, ref[k], ref['e' + k], k)


@pytest.mark.gpu
@pytest.mark.parametrize('n', [6, 140])
@pytest.mark.parametrize('sizes', [(1e30, 1e-20), (1e-20, 1e30), (1e-37, 1e8, 1e-30, 1e30, 1, 1e-12, 1e-37, 1e30), (2.0 ** 49, 1e-25)])
def test_fc_logreg_weights_of_any_sizes_stay_in_range(sizes, n):
    """Groups of classes whose weights differ by up to 2^220, in both orders: the sum over the classes is neither infinite nor lost."""
    d, v = 40, 64 * len(sizes)
    w, x, b, lab = fcl_data(d, v, n, 38, lean=0)
    rng = np.random.default_rng(39)
    w *= np.repeat(np.float32(sizes), 64)[:, None]
    x /= np.float32(max(sizes))
    ref = fcl_ref(w, x, b, lab, 0.5)
    st, lp, ok, dx, dw, db, _ = fcl_run(w, x, b, lab, 0.5)
    check_forward(ref, st, lp, ok)
    for got, k in ((dx, 'dx'), (db, 'db')):
        within(got, ref[k], ref['e' + k], k)
    within(dw, ref['dw'], ref['edw'] + 2.0 ** -126, 'dw')  # (products down to 1e-38: what is below the smallest normal number may be zero)
    # and where the large classes are out, by a bias of -inf or by one that leaves no probability: the small ones' sum and nothing else
    large = np.repeat(np.float32(sizes), 64) >= 1
    lab2 = rng.choice(np.flatnonzero(~large), n).astype(np.float32)
    for out in (-np.inf, -1000):
        b2 = np.where(large, np.float32(out), b)
        ref = fcl_ref(np.where(np.isneginf(b2)[:, None], 0, w), x, b2, lab2, 0.5)
        dx = fcl_run(w, x, b2, lab2, 0.5)[3]
        within(dx, ref['dx'], ref['edx'] + 2.0 ** -126, 'dx of small weights')


@pytest.mark.gpu
@pytest.mark.parametrize('d,v,n', [(36, 500, 6), (36, 500, 64), (40, 33000, 20), (40, 700, 140), (160, 10575, 509), (96, 10575, 509), (300, 70000, 70), (64, 3000, 1025), (20, 300, 4500)])
def test_fc_logreg_classes_that_no_case_comes_near(d, v, n):
    """Probabilities from 1 down to 2^-90: every class's weight gradient is right relative to itself, beside labels' classes and others, and
    where a class is near some cases and far from others (feature 0 changes its sign every 64 to 192 cases)."""
    rng = np.random.default_rng(45)
    w = (rng.standard_normal((v, d)) / np.sqrt(d)).astype(np.float32)
    x = rng.standard_normal((d, n)).astype(np.float32)
    x[0] = np.where(np.arange(n) // 64 % 5 < 2, 1, -1)
    w[:, 0] = rng.choice([-10, 0, 10], v)
    b = (-np.log(2) * 52 * rng.random(v)).astype(np.float32)
    near = rng.permutation(v)[:max(v // 8, 4)]
    b[near], w[near, 0] = 0, 0
    lab = rng.choice(near, n).astype(np.float32)
    lab[n - n // 7:] = -1
    ref = fcl_ref(w, x, b, lab, 0.5)
    largest = np.abs(ref['dz']).max(1)
    assert (largest < 2.0 ** -45).sum() > v // 20 and largest[largest > 0].min() > 2.0 ** -92
    st, lp, ok, dx, dw, db, cost = fcl_run(w, x, b, lab, 0.5)
    check_forward(ref, st, lp, ok)
    for got, k in ((dx, 'dx'), (dw, 'dw'), (db, 'db')):
        within(got, ref[k], ref['e' + k], k)


@pytest.mark.gpu
@pytest.mark.parametrize('d,v,n', [(36, 500, 64), (40, 700, 140), (160, 10575, 509)])
def test_fc_logreg_nothing_of_an_earlier_call_stays(d, v, n):
    """One workspace, eager and in a replayed graph: classes far from every case, then near ones, then far again -- the bits of a workspace of
    one's own."""
    w, x, b, lab = fcl_data(d, v, n, 47)
    far = np.where(np.arange(v) % 2, np.float32(-30), np.float32(0))
    lab = np.floor(lab / 2) * 2  # (classes at 0)
    ws, size = need('mcn_fc_logreg_workspace_bytes', d, v, n, 1)
    kw, kx, kl, kb = dev(w), dev(x), dev(lab), dev(b)
    outs = [Out(s) for s in ((2, n), (n,), (n,), (d, n), (v, d), (v,))]
    stream = C.c_void_p()
    call('mcn_stream_create', C.byref(stream))

    def step():
        call('mcn_fc_logreg_cost', kw, kx, kb, kl, *outs[:3], d, v, n, None, ws, size, stream)
        call('mcn_fc_logreg_grad', kw, kx, kb, kl, outs[0], *outs[3:], d, v, n, 0.5, 0.0, 0.0, 1.0, 0.0, 1.0, ws, size, stream)

    want = {False: fcl_run(w, x, b, lab, 0.5), True: fcl_run(w, x, b + far, lab, 0.5)}
    step()
    exe = C.c_void_p()
    call('mcn_stream_sync', stream)
    call('mcn_graph_begin_capture', stream)
    step()
    call('mcn_graph_end_capture', stream, C.byref(exe), None)
    for k, distant in enumerate((True, False, True, True, False, False, True)):
        kb.upload(b + far if distant else b)
        call('mcn_device_sync')
        call('mcn_graph_launch', exe, stream) if k % 3 else step()
        call('mcn_stream_sync', stream)
        for o, a in zip(outs, want[distant]):
            assert np.array_equal(o.get(), a), k
    call('mcn_graph_destroy', exe)
    call('mcn_stream_destroy', stream)


@pytest.mark.gpu
@pytest.mark.parametrize('d,v,n', [(12, 30, 9), (40, 150, 66)])
def test_fc_logreg_gradient_against_differences(d, v, n):
    """d sum(log p) along random directions (central differences of the float64 formula, step 1e-4: 1e-6 of the magnitudes)."""
    w, x, b, lab = fcl_data(d, v, n, 17, padded=2)
    _, _, _, dx, dw, db, _ = fcl_run(w, x, b, lab)
    ref = fcl_ref(w, x, b, lab, 1.0)
    rng = np.random.default_rng(6)
    base = [a.astype(np.float64) for a in (x, w, b)]
    for k, (got, e) in enumerate(((dx, 'edx'), (dw, 'edw'), (db, 'edb'))):
        dirn = rng.standard_normal(got.shape)
        h = 1e-4

        def value(s):
            p = [a + s * dirn if i == k else a for i, a in enumerate(base)]
            z = p[1] @ p[0] + p[2][:, None]
            top = z.max(0)
            lse = top + np.log(np.exp(z - top).sum(0))
            return sum(z[int(lab[c]), c] - lse[c] for c in range(n) if lab[c] >= 0)
        want = (value(h) - value(-h)) / (2 * h)
        assert abs((got * dirn).sum() - want) <= (ref[e] * np.abs(dirn)).sum() + 1e-6 * np.abs(got * dirn).sum()


# ------------------------------------------------------------------------------------------------------------- together
def head_ref(x, gain, bias, w, b, lab, keep, p, coeff):
    y, mean, r = norm_ref(x, gain, bias)
    s = keep / (1 - float(np.float32(p)))
    ref = fcl_ref(w, y * s, b, lab, coeff)
    dy = ref['dx'] * s
    dx, dgain, dbias = undo_ref(dy, x, gain, mean, r)
    return ref, dx, dgain, dbias


@pytest.mark.gpu
@pytest.mark.parametrize('captured', [False, True])
@pytest.mark.parametrize('n', [96, 24])
def test_head_together(captured, n):
    """norm -> dropout -> classifier cost and back, on a stream of its own: eager, and as a graph that is replayed with new masks
    between the program's own eager work.  Six stages, each with sums of at most 900 terms (sum_err(900) = 1.5e-5 of the magnitudes):
    1e-4 of the largest value."""
    f, v, p, coeff = 160, 900, 0.4, 1.0 / n
    x, gain, bias, _ = norm_data(f, n, 21)
    w, _, b, lab = fcl_data(f, v, n, 22)
    stream = C.c_void_p()
    call('mcn_stream_create', C.byref(stream))
    kx, kg, kb, kw, kbb, kl = (dev(a) for a in (x, gain, bias, w, b, lab))
    y, st, drop = Out((f, n)), Out((2, n)), Out((f, n))
    cst, lp, ok = Out((2, n)), Out((n,)), Out((n,))
    dd, dw, db, dn, dg, dbi = Out((f, n)), Out((v, f)), Out((v,)), Out((f, n)), Out((f,)), Out((f,))
    counter = capi.DeviceBuffer(array=np.array([100], np.uint64))
    sizes = [need('mcn_layer_norm_workspace_bytes', f, n), need('mcn_layer_norm_undo_workspace_bytes', f, n),
             need('mcn_fc_logreg_workspace_bytes', f, v, n, 1)]
    (w1, s1), (w2, s2), (w3, s3) = sizes

    def step():
        call('mcn_counter_add', counter.ptr, 1, stream)
        call('mcn_layer_norm', kx, kg, kb, y, st, f, n, EPS, w1, s1, stream)
        call('mcn_dropout', y, drop, f * n, p, 99, 0, counter.ptr, 0.0, 1.0, stream)
        call('mcn_fc_logreg_cost', kw, drop, kbb, kl, cst, lp, ok, f, v, n, None, w3, s3, stream)
        call('mcn_fc_logreg_grad', kw, drop, kbb, kl, cst, dd, dw, db, f, v, n, coeff, 0.0, 0.0, 1.0, 0.0, 1.0, w3, s3, stream)
        call('mcn_dropout', dd, dd, f * n, p, 99, 0, counter.ptr, 0.0, 1.0, stream)
        call('mcn_layer_norm_undo', dd, kx, kg, st, dn, dg, dbi, f, n, 0.0, 1.0, 0.0, 1.0, 0.0, 1.0, w2, s2, stream)

    exe = C.c_void_p()
    if captured:
        step()  # once eagerly, as a program would
        call('mcn_stream_sync', stream)
        call('mcn_graph_begin_capture', stream)
        step()
        call('mcn_graph_end_capture', stream, C.byref(exe), None)
    for k in range(4):
        if captured:
            call('mcn_graph_launch', exe, stream)
        else:
            step()
        call('mcn_stream_sync', stream)
        number = 101 + k + (1 if captured else 0)
        keep = kept(f * n, p, 99, number).reshape(f, n)
        ref, wx, wg, wb = head_ref(x.astype(np.float64), gain.astype(np.float64), bias.astype(np.float64), w, b, lab, keep, p, coeff)
        for got, want, what in ((lp, ref['logp'], 'logp'), (dw, ref['dw'], 'dw'), (db, ref['db'], 'db'), (dn, wx, 'dx'), (dg, wg, 'dgain'), (dbi, wb, 'dbias')):
            within(got.get(), want, 1e-4 * np.abs(want).max(), '%s of step %d' % (what, k))
        # eager work of the program between the replays
        other = Out((f, n))
        call('mcn_layer_norm', kx, None, None, other, None, f, n, EPS, w1, s1, None)
        call('mcn_device_sync')
    if captured:
        call('mcn_graph_destroy', exe)
    call('mcn_stream_destroy', stream)


@pytest.mark.gpu
@pytest.mark.parametrize('d,v,n', [(160, 4213, 1), (160, 1000, 128), (5000, 300, 130)])
def test_head_two_at_once(d, v, n):
    """The same calls on two streams at once, each with workspaces of its own: the bits of one alone."""
    w, x, b, lab = fcl_data(d, v, n, 41)
    g, gain, bias, _ = norm_data(d, n, 42)
    kw, kx, kb, kl, kg, kgain, kbias = (dev(a) for a in (w, x, b, lab, g, gain, bias))

    class Side:
        def __init__(self):
            self.stream = C.c_void_p()
            call('mcn_stream_create', C.byref(self.stream))
            self.ws = [need('mcn_fc_logreg_workspace_bytes', d, v, n, 1), need('mcn_layer_norm_workspace_bytes', d, n),
                       need('mcn_layer_norm_undo_workspace_bytes', d, n)]
            self.o = [Out(s) for s in ((d, n), (2, n), (2, n), (n,), (n,), (d, n), (v, d), (v,), (d, n), (d,), (d,))]

        def run(self):
            (cw, cs), (fw, fs), (uw, us) = self.ws
            y, st, cst, lp, ok, dx, dw, db, dn, dg, dbi = self.o
            s = self.stream
            call('mcn_layer_norm', kx, kgain, kbias, y, st, d, n, EPS, fw, fs, s)
            call('mcn_fc_logreg_cost', kw, y, kb, kl, cst, lp, ok, d, v, n, None, cw, cs, s)
            call('mcn_fc_logreg_grad', kw, y, kb, kl, cst, dx, dw, db, d, v, n, 0.5, 0.0, 0.0, 1.0, 0.0, 1.0, cw, cs, s)
            call('mcn_layer_norm_undo', kg, kx, kgain, st, dn, dg, dbi, d, n, 0.0, 1.0, 0.0, 1.0, 0.0, 1.0, uw, us, s)

    one, two = Side(), Side()
    one.run()
    call('mcn_device_sync')
    want = [o.get() for o in one.o]
    assert all(np.isfinite(a).all() for a in want)
    for _ in range(3):
        for _ in range(4):
            one.run()
            two.run()
        call('mcn_device_sync')
        for side in (one, two):
            for o, a in zip(side.o, want):
                assert np.array_equal(o.get(), a)
    for side in (one, two):
        call('mcn_stream_destroy', side.stream)


# ------------------------------------------------------------------------------------------------------------- beyond 32 bits
class Huge(capi.DeviceBuffer):
    """`count` zeros, of which single stretches are set and read."""

    def __init__(self, count):
        super().__init__(nbytes=count * 4)
        self.zero()

    def put(self, at, a):
        a = np.ascontiguousarray(a, np.float32)
        call('mcn_h2d', self.ptr + at * 4, a.ctypes.data, a.nbytes, None)
        call('mcn_device_sync')

    def take(self, at, count):
        out = np.empty(count, np.float32)
        call('mcn_device_sync')
        call('mcn_d2h', out.ctypes.data, self.ptr + at * 4, out.nbytes, None)
        call('mcn_device_sync')
        return out


@pytest.mark.gpu
def test_dropout_beyond_32_bits():
    n, tail = (1 << 32) + 1003, 4096
    at = n - tail - (n - tail) % 4
    count = n - at
    big = Huge(n)
    x = np.random.default_rng(51).standard_normal(count).astype(np.float32)
    big.put(at, x)
    call('mcn_dropout', big, big, n, 0.4, 5, 6, None, 0.0, 1.0, None)
    keep = philox_words(count, 5, 6, first_quad=at // 4) >= np.uint32(int(float(np.float32(0.4)) * 2 ** 32))
    want = np.where(keep, x / (1 - float(np.float32(0.4))), 0)
    within(big.take(at, count), want, 2 * U * np.abs(want), 'tail')
    assert not big.take(0, 1 << 20).any()


@pytest.mark.gpu
@pytest.mark.parametrize('f,n', [(300, 14500001), (66000, 65541)])  # whole columns in registers, ranges of rows
def test_layer_norm_beyond_32_bits(f, n):
    """Two columns at the very end and one at the start hold something (the last row, and the first, of all columns too)."""
    assert f * n > 1 << 32
    rng = np.random.default_rng(52)
    rows = {r: rng.standard_normal(n).astype(np.float32) for r in (0, f - 1)}
    gain, bias = (rng.standard_normal(f).astype(np.float32) for _ in range(2))
    big, dx = Huge(f * n), Huge(f * n)
    for r, a in rows.items():
        big.put(r * n, a)
    st = Out((2, n))
    ws, size = need('mcn_layer_norm_workspace_bytes', f, n)
    kg, kb = dev(gain), dev(bias)
    call('mcn_layer_norm', big, kg, kb, dx, st, f, n, EPS, ws, size, None)
    a = np.stack([rows[0], rows[f - 1]]).astype(np.float64)
    mean = a.sum(0) / f
    r = 1 / np.sqrt((((a - mean) ** 2).sum(0) + (f - 2) * mean ** 2) / f + EPS)
    got = st.get()
    within(got[0], mean, (sum_err(f) + 4 * U) * np.abs(a).sum(0) / f + 1e-12, 'means')
    within(got[1], r, (sum_err(f) + 16 * U) * r, 'r')
    bound = lambda k, v: np.abs(gain[k]) * (sum_err(f) + 32 * U) * (np.abs(v) * r) + 4 * U * np.abs(bias[k]) + 1e-12  # noqa: E731
    for k, v in ((0, a[0] - mean), (f - 2, -mean), (f - 1, a[1] - mean)):
        within(dx.take(k * n, n), gain[k] * (v * r) + bias[k], bound(k, np.abs(v) + np.abs(a).sum(0) / f), 'row %d' % k)
    # backward: the outputs' gradient is the input itself, its target the matrix of outputs
    dg, db = Out((f,)), Out((f,))
    ws, size = need('mcn_layer_norm_undo_workspace_bytes', f, n)
    grad = Huge(f * n)
    for k, v in rows.items():
        grad.put(k * n, v)
    call('mcn_layer_norm_undo', grad, big, kg, st, dx, dg, db, f, n, 0.0, 1.0, 0.0, 1.0, 0.0, 1.0, ws, size, None)
    mu, rs = got.astype(np.float64)
    xh = (a - mu) * rs
    h = np.stack([gain[0] * a[0], gain[f - 1] * a[1]]).astype(np.float64)
    s1, s2 = h.sum(0) / f, (h * xh).sum(0) / f
    for i, k in enumerate((0, f - 1)):
        want = rs * (h[i] - s1 - xh[i] * s2)
        within(dx.take(k * n, n), want, (sum_err(f) + 64 * U) * rs * (np.abs(h[i]) + np.abs(h).sum(0) / f + np.abs(xh[i]) * np.abs(h * xh).sum(0) / f) + 1e-12, 'dx of row %d' % k)
        assert abs(dg.get()[k] - (a[i] * xh[i]).sum()) <= (sum_err(n) + 16 * U) * (np.abs(a[i]) * (np.abs(a[i]) + np.abs(mu)) * rs).sum()
        assert abs(db.get()[k] - a[i].sum()) <= (sum_err(n) + 4 * U) * np.abs(a[i]).sum()
    assert not dg.get()[1:f - 1].any() and not db.get()[1:f - 1].any()


@pytest.mark.gpu
@pytest.mark.parametrize('n', [3, 70])
def test_fc_logreg_beyond_32_bits(n):
    """The most classes there can be; the weights of the first and the last two are not zero."""
    d, v, coeff = 260, 1 << 24, 0.5
    assert d * v > 1 << 32
    rng = np.random.default_rng(53)
    some = np.array([0, v - 2, v - 1])
    ws_rows = rng.standard_normal((3, d)).astype(np.float32)
    x = rng.standard_normal((d, n)).astype(np.float32)
    lab = some[np.arange(n) % 3].astype(np.float32)
    w, dw = Huge(d * v), Huge(d * v)
    for r, a in zip(some, ws_rows):
        w.put(int(r) * d, a)
    st, lp, ok, dx, db = Out((2, n)), Out((n,)), Out((n,)), Out((d, n)), Out((v,))
    ws, size = need('mcn_fc_logreg_workspace_bytes', d, v, n, 1)
    kx, kl = dev(x), dev(lab)
    call('mcn_fc_logreg_cost', w, kx, None, kl, st, lp, ok, d, v, n, None, ws, size, None)
    call('mcn_fc_logreg_grad', w, kx, None, kl, st, dx, dw, db, d, v, n, coeff, 0.0, 0.0, 1.0, 0.0, 1.0, ws, size, None)
    w64, x64 = ws_rows.astype(np.float64), x.astype(np.float64)
    z = w64 @ x64
    top = np.maximum(z.max(0), 0)
    e = np.exp(z - top)
    tot = (v - 3) * np.exp(-top) + e.sum(0)
    ez = (sum_err(d) + 4 * U) * (np.abs(w64) @ np.abs(x64)).max(0)
    er = 2 * ez + sum_err(v) + 16 * U
    zl = z[np.arange(n) % 3, np.arange(n)]
    within(lp.get(), zl - top - np.log(tot), 2 * er + 4 * U * np.abs(zl - top - np.log(tot)), 'logp')
    dz = -e / tot
    dz[np.arange(n) % 3, np.arange(n)] += 1
    dz *= coeff
    edz = e / tot * er + 4 * U * np.abs(dz) + 2.0 ** -43
    within(dx.get(), w64.T @ dz, np.abs(w64).T @ edz + 16 * U * np.abs(w64).T @ np.abs(dz), 'dx')
    rest = -coeff * np.exp(-top) / tot  # dz of every other class
    for i, r in enumerate(some):
        within(dw.take(int(r) * d, d), x64 @ dz[i], np.abs(x64) @ edz[i] + (sum_err(n) + 2 * U) * np.abs(x64) @ np.abs(dz[i]), 'dw of class %d' % r)
        assert abs(db.get()[r] - dz[i].sum()) <= edz[i].sum() + sum_err(n) * np.abs(dz[i]).sum()
    within(dw.take((v - 3) * d, d), x64 @ rest, np.abs(x64) @ (np.abs(rest) * er + 2.0 ** -43) + (sum_err(n) + 2 * U) * np.abs(x64) @ np.abs(rest), 'dw before them')
