"""The preference loss on packed pairs and the sequences' log-probabilities against the formula in
64 bits.

Tolerances (u = 2^-24): a row's sum of n exponentials is off by at most (n + 4) u relative (the base-2
exponential is within two units of its value) and 3 |z - max| u more (z - max is rounded, multiplied by a
rounded log2(e), and rounded again), so its log-probability by (n + 4 + 3 R) u and 2 u R with R the largest |z - max|; a sequence's log-probability by the sum of its rows' and one rounding.
x is off by beta times its two sequences' bounds, a factor by beta / pairs times a quarter of that (the
sigmoid's slope) and a rounding, a gradient element by the factor's and the softmax's error
(its own exponential's 3 R u and its sum's 3 R u).
"""
import numpy as np
import pytest

import freeml_amd as fh
from graphs import Captured

U = 2.0**-24
MARK = np.float32(-7.5)


def inputs(lens, vocab, seed, std=2.0, ignored=0.3, extra=(0, 0)):
    r = np.random.default_rng(seed)
    off = np.cumsum([extra[0]] + list(lens)).astype(np.int32)
    rows = int(off[-1]) + extra[1]
    z = (std * r.standard_normal((rows, vocab))).astype(np.float32)
    t = r.integers(0, vocab, rows).astype(np.float32)
    t[r.random(rows) < ignored] = -1.0
    ref = np.array([-n * 0.7 * np.log(vocab) for n in lens] + 3 * r.standard_normal(len(lens))).astype(np.float32)
    return off, rows, z, t, ref


def reference(off, z, t, ref, beta, smoothing):
    z64 = z.astype(np.float64)
    top = z64.max(1, keepdims=True)
    e = np.exp(z64 - top)
    soft = e / e.sum(1, keepdims=True)
    V = z.shape[1]
    ids = np.where((t > -1) & (t < V), np.trunc(t), -1).astype(np.int64)
    ok = ids >= 0
    row = np.where(ok, (z64 - top)[np.arange(len(t)), np.maximum(ids, 0)] - np.log(e.sum(1)), 0.0)
    R = np.where(np.isfinite(z64), top - z64, 0.0).max(1)
    b_row = np.where(ok, (V + 4 + 5 * R) * U, 0.0)
    lp = np.array([row[a:b].sum() for a, b in zip(off, off[1:])])
    b_lp = np.array([b_row[a:b].sum() for a, b in zip(off, off[1:])])
    out = dict(lp=lp, b_lp=b_lp + np.abs(lp) * U)
    if ref is None:
        return out
    P = len(lp) // 2
    ratio = lp - ref.astype(np.float64)
    x = beta * (ratio[0::2] - ratio[1::2])
    b_x = beta * (b_lp[0::2] + b_lp[1::2])
    loss = (1 - smoothing) * np.logaddexp(0, -x) + (smoothing * np.logaddexp(0, x) if smoothing else 0.0)
    with np.errstate(over="ignore"):
        f = beta / P * ((1 - smoothing) / (1 + np.exp(x)) - smoothing / (1 + np.exp(-x)))
    grad, b_grad = np.full(z.shape, float(MARK)), np.zeros(z.shape)
    onehot = np.zeros(z.shape)
    onehot[np.nonzero(ok)[0], ids[ok]] = 1.0
    for s, (a, b) in enumerate(zip(off, off[1:])):
        sign = f[s // 2] * (1 if s % 2 == 0 else -1)
        grad[a:b] = sign * (onehot - soft)[a:b] * ok[a:b, None]
        b_grad[a:b] = ((beta / P * b_x[s // 2] / 4 + 4 * U * abs(sign)) * np.abs((onehot - soft)[a:b]) +
                       abs(sign) * (soft * ((V + 8 + 6 * R)[:, None] * U) + 2 * U * onehot)[a:b]) * ok[a:b, None]
    out.update(loss=loss.mean(), b_loss=b_x.mean() + np.abs(loss).mean() * 4 * U, grad=grad, b_grad=b_grad, x=x)
    return out


def run(off, rows, z, t, ref, beta=0.1, smoothing=0.0, in_place=False, loss=True, logp=True, grad=True, shift=0):
    dev = fh.DeviceArray.from_host
    V, n = z.shape[1], len(off) - 1

    def place(a):
        d = dev(np.concatenate([np.full(shift, MARK, np.float32), np.asarray(a, np.float32).ravel()]))
        return d, d.at(shift)

    dz, pz = place(z)
    dg, pg = (dz, pz) if in_place else place(np.full(z.shape, MARK, np.float32))
    dt, dl, dp, dr, do = dev(t), dev(np.full(1, MARK)), dev(np.full(n, MARK)), dev(ref), dev(off)
    ws = dev(np.full(max(2, fh.preference_workspace(rows, n)), np.nan, np.float32))
    fh.preference_logits(pg if grad else 0, dl.ptr if loss else 0, dp.ptr if logp else 0, ws.ptr, dt.ptr, pz, do.ptr, dr.ptr, V, rows,
                         n // 2, beta, smoothing)
    return dg.numpy()[shift:].reshape(z.shape), dl.numpy()[0], dp.numpy()


def close(got, ref, bound, what):
    far = np.abs(np.asarray(got, np.float64) - ref) - bound - np.abs(ref) * U - 2.0**-126
    assert np.all(far <= 0), f"{what}: worst {np.max(far)} beyond its bound"


CASES = [([3, 4], 5), ([1, 1], 1), ([20, 7, 0, 5], 65), ([300, 2, 9, 9], 257), ([40, 33], 1000), ([5, 6], 4099), ([3, 2], 32003),
         ([2, 3], 50304), ([2, 1], 70001), ([0, 0, 4, 4], 64), ([1] * 40, 33), ([17, 1200], 48)]


@pytest.mark.gpu
@pytest.mark.parametrize("smoothing", [0.0, 0.2])
@pytest.mark.parametrize("lens,vocab", CASES)
def test_loss_and_gradient(lens, vocab, smoothing):
    print(f"pairs {lens[:6]} vocab {vocab} smoothing {smoothing}", flush=True)
    off, rows, z, t, ref = inputs(lens, vocab, seed=vocab, extra=(1, 2))
    r = reference(off, z, t, ref, np.float64(np.float32(0.1)), np.float64(np.float32(smoothing)))
    grad, loss, logp = run(off, rows, z, t, ref, smoothing=smoothing)
    close(logp, r["lp"], r["b_lp"], "logp")
    close(loss, r["loss"], r["b_loss"], "loss")
    close(grad, r["grad"], r["b_grad"], "grad")


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [65, 1001, 4100, 50304])
@pytest.mark.parametrize("shift", [0, 1, 2])
def test_gradient_in_place_and_any_alignment(vocab, shift):
    """In place, and at any alignment: the same bits."""
    off, rows, z, t, ref = inputs([6, 5, 2, 9], vocab, seed=1, extra=(0, 3))
    a = run(off, rows, z, t, ref)[0]
    b = run(off, rows, z, t, ref, in_place=True, shift=shift)[0]
    n = off[-1]
    np.testing.assert_array_equal(a[:n], b[:n])
    np.testing.assert_array_equal(b[n:], z[n:])
    r = reference(off, z, t, ref, np.float64(np.float32(0.1)), 0.0)
    close(a, r["grad"], r["b_grad"], "grad")


@pytest.mark.gpu
@pytest.mark.parametrize("lens,vocab", [([4], 65), ([3, 0, 7], 50304), ([200] * 9, 131), ([1000], 2048)])
def test_sequence_logprobs(lens, vocab):
    off, rows, z, t, _ = inputs(lens, vocab, seed=2, extra=(2, 1))
    dev = fh.DeviceArray.from_host
    dz, dt, do, dp = dev(z), dev(t), dev(off), dev(np.full(len(lens), MARK))
    ws = dev(np.full(fh.preference_workspace(rows, len(lens)), np.nan, np.float32))
    fh.sequence_logprobs(dp.ptr, ws.ptr, dt.ptr, dz.ptr, do.ptr, vocab, rows, len(lens))
    r = reference(off, z, t, None, 0, 0)
    close(dp.numpy(), r["lp"], r["b_lp"], "logp")


@pytest.mark.gpu
def test_outputs_that_are_not_asked_for():
    off, rows, z, t, ref = inputs([6, 5], 90, seed=3)
    grad, loss, logp = run(off, rows, z, t, ref)
    for which in ("grad", "loss", "logp"):
        g, l, p = run(off, rows, z, t, ref, **{w: w == which for w in ("grad", "loss", "logp")})
        for name, got, full in (("grad", g, grad), ("loss", l, loss), ("logp", p, logp)):
            np.testing.assert_array_equal(got, full if name == which else MARK)


@pytest.mark.gpu
def test_gradient_is_the_descent_direction():
    """Central differences of the loss: a step of h along a direction changes it by -h grad . direction.
    The loss is off by b_loss either way, so the quotient by b_loss / h; the third-order term is below 1e-3 of it."""
    off, rows, z, t, ref = inputs([4, 5, 3, 6], 40, seed=4, ignored=0.2)
    grad = run(off, rows, z, t, ref, beta=0.5)[0]
    r = np.random.default_rng(0)
    d = r.choice([-1.0, 1.0], z.shape).astype(np.float32)
    d[off[-1]:] = 0
    h = 2.0**-6
    up, dn = (run(off, rows, (z + s * h * d).astype(np.float32), t, ref, beta=0.5)[1] for s in (1, -1))
    slope = -np.sum(grad.astype(np.float64) * d)
    b = reference(off, z, t, ref, 0.5, 0.0)["b_loss"]
    assert abs((float(up) - float(dn)) / (2 * h) - slope) <= b / h + 2e-3 * np.sum(np.abs(grad)), slope


@pytest.mark.gpu
def test_equal_pairs_cancel():
    """The same logits and targets chosen and rejected: x = 0, loss = log 2 and gradients of opposite sign."""
    _, _, z, t, _ = inputs([5, 5], 77, seed=5)
    z[5:], t[5:] = z[:5], t[:5]
    grad, loss, logp = run(np.array([0, 5, 10], np.int32), 10, z, t, np.zeros(2, np.float32), beta=0.3)
    assert logp[0] == logp[1] and abs(loss - np.log(2)) <= 2 * U
    np.testing.assert_array_equal(grad[:5], -grad[5:])


@pytest.mark.gpu
def test_extremes():
    """Margins that saturate the sigmoid, logits of -infinity off the target (no weight, no gradient), large logits."""
    off, rows, z, t, _ = inputs([3, 3], 50, seed=6, ignored=0.0)
    for ref in ([-3e4, 3e4], [3e4, -3e4]):
        ref = np.array(ref, np.float32)
        grad, loss, _ = run(off, rows, z, t, ref, beta=1.0)
        r = reference(off, z, t, ref, 1.0, 0.0)
        close(loss, r["loss"], r["b_loss"], "loss")
        assert np.all(np.isfinite(grad))
    z2 = z.copy()
    z2[:, ::2] = -np.inf
    t2 = np.full_like(t, 3.0)
    grad, loss, logp = run(off, rows, z2, t2, np.zeros(2, np.float32))
    assert np.all(np.isfinite(logp)) and np.isfinite(loss) and np.all(grad[:, ::2] == 0) and np.all(np.isfinite(grad))
    big = (z * 1e30).astype(np.float32)
    t3 = np.argmax(big, 1).astype(np.float32)
    grad, loss, logp = run(off, rows, big, t3, np.zeros(2, np.float32))
    assert np.all(logp == 0) and abs(loss - np.log(2)) <= 2 * U and np.all(np.abs(grad) <= U)


@pytest.mark.gpu
def test_targets_outside_the_vocabulary_do_not_count():
    off, rows, z, t, ref = inputs([4, 4], 30, seed=7, ignored=0.0)
    t[1], t[2], t[5], t[6] = 30.0, np.nan, -2.0, 3e9
    t[0], t[4] = 7.75, -0.5  # truncated: 7 and 0
    grad, loss, logp = run(off, rows, z, t, ref)
    r = reference(off, z, t, ref, np.float64(np.float32(0.1)), 0.0)
    close(logp, r["lp"], r["b_lp"], "logp")
    close(grad, r["grad"], r["b_grad"], "grad")


@pytest.mark.gpu
def test_captured_and_replayed():
    off, rows, z, t, ref = inputs([30, 20, 7, 40], 500, seed=8)
    dev = fh.DeviceArray.from_host
    dz, dg, dt, do, dr = dev(z), dev(np.zeros_like(z)), dev(t), dev(off), dev(ref)
    dl, dp = dev(np.zeros(1, np.float32)), dev(np.zeros(4, np.float32))
    ws = dev(np.zeros(fh.preference_workspace(rows, 4), np.float32))

    def calls():
        fh.preference_logits(dg.ptr, dl.ptr, dp.ptr, ws.ptr, dt.ptr, dz.ptr, do.ptr, dr.ptr, 500, rows, 2)

    calls()
    g = Captured(calls)
    r = np.random.default_rng(1)
    for _ in range(4):
        dz.upload(r.standard_normal(z.shape).astype(np.float32))
        got = []
        for replay in (False, True):
            for d in (dg, dl, dp):
                d.upload(np.full(d.shape, MARK, np.float32))
            if replay:
                g.replay()
            else:
                calls()
            got.append([d.numpy() for d in (dg, dl, dp)])
        for a, b in zip(*got):
            np.testing.assert_array_equal(a, b)


# ---- refusals (no device needed) -----------------------------------------------------------------

@pytest.mark.parametrize("over", [dict(ws=0), dict(ws=4), dict(target=0), dict(logits=0), dict(off=0), dict(ref_logp=0), dict(vocab=0),
                                  dict(vocab=2**24 + 1), dict(rows=2**23 + 1), dict(pairs=0), dict(pairs=2**23 + 1), dict(beta=0.0),
                                  dict(beta=-1.0), dict(beta=float("nan")), dict(beta=float("inf")), dict(smoothing=-0.1), dict(smoothing=0.6),
                                  dict(smoothing=float("nan")), dict(grad=0, loss=0, logp=0)], ids=str)
def test_refusals(over):
    a = dict(grad=8, loss=8, logp=8, ws=8, target=8, logits=8, off=8, ref_logp=8, vocab=10, rows=4, pairs=1, beta=0.1, smoothing=0.0)
    with pytest.raises(fh.FreeMLHipError) as e:
        fh.preference_logits(**{**a, **over})
    assert e.value.code == -1


@pytest.mark.parametrize("over", [dict(logp=0), dict(ws=0), dict(target=0), dict(logits=0), dict(off=0), dict(vocab=0), dict(n_seq=2**24 + 1)], ids=str)
def test_refusals_of_logprobs(over):
    a = dict(logp=8, ws=8, target=8, logits=8, off=8, vocab=10, rows=4, n_seq=2)
    with pytest.raises(fh.FreeMLHipError) as e:
        fh.sequence_logprobs(**{**a, **over})
    assert e.value.code == -1
