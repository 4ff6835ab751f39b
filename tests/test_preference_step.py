"""Preference tuning from end to end through the operator API: a tied-embedding layer of grouped-head
attention on packed pairs, the reference model's log-probabilities, the loss and its gradients down
to every weight, an AdamW step over all of them, and the tuned model continuing a sequence one token
at a time over a key/value cache.  Against numpy in 64 bits, whose gradients are checked against
differences of its own loss.

Tolerances: the longest chain of sums here (embedding gradient: logits, loss, products, attention,
products) has about 6 sums of up to 600 terms; each rounds by at most 600 x 2^-24 = 3.6e-5 of its terms'
absolute values, and terms of both signs grow that by the ratio of absolute to net sum, below 5 here: the
2-norm of an error is below 6 x 5 x 3.6e-5 / sqrt(600), the roundings being independent: 5e-5.
"""
import numpy as np
import pytest

import freeml_amd as fh

V, C, H, HK, D = 97, 48, 6, 2, 16
W = (H + 2 * HK) * D
LENS = [23, 31, 9, 40]  # two pairs, chosen and rejected
ROWS = sum(LENS)
OFF = np.cumsum([0] + LENS).astype(np.int32)
SCALE = D**-0.5
TOL = 5e-5
LR, B1, B2, EPS, WD = 1e-3, 0.9, 0.999, 1e-8, 0.01


def weights(seed):
    r = np.random.default_rng(seed)
    f = lambda *s, std=0.2: (std * r.standard_normal(s)).astype(np.float32)  # noqa: E731
    return dict(emb=f(V, C, std=0.5), qkv=f(C, W), proj=f(H * D, C))


def data():
    r = np.random.default_rng(1)
    ids = r.integers(0, V, ROWS)
    target = np.roll(ids, -1).astype(np.float32)
    for a, b in zip(OFF, OFF[1:]):
        target[a:a + 5] = -1  # the prompt
        target[b - 1] = -1    # nothing follows
    return ids, target


# ---- numpy in 64 bits -----------------------------------------------------------------------------

def np_forward(w, ids):
    w = {k: x.astype(np.float64) for k, x in w.items()}
    x = w["emb"][ids]
    qkv = x @ w["qkv"]
    y, ps = np.zeros((ROWS, H * D)), {}
    for s, (a, b) in enumerate(zip(OFF, OFF[1:])):
        for h in range(H):
            q, k, v = np_heads(qkv[a:b], h)
            sc = np.where(np.tri(b - a, dtype=bool), q @ k.T * SCALE, -np.inf)
            p = np.exp(sc - sc.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            ps[s, h] = p
            y[a:b, h * D:(h + 1) * D] = p @ v
    hid = x + y @ w["proj"]
    return dict(w=w, x=x, qkv=qkv, y=y, ps=ps, hid=hid, logits=hid @ w["emb"].T)


def np_heads(qkv, h):
    at = [h * D, (H + h // (H // HK)) * D, (H + HK + h // (H // HK)) * D]
    return (qkv[:, i:i + D] for i in at)


def np_logp(logits, target):
    z = logits - logits.max(1, keepdims=True)
    lp = z - np.log(np.exp(z).sum(1, keepdims=True))
    row = np.where(target >= 0, lp[np.arange(ROWS), np.maximum(target, 0).astype(int)], 0)
    return np.exp(lp), np.array([row[a:b].sum() for a, b in zip(OFF, OFF[1:])])


def np_loss(logits, target, ref, beta):
    soft, lp = np_logp(logits, target)
    x = beta * ((lp - ref)[0::2] - (lp - ref)[1::2])
    f = beta / len(x) / (1 + np.exp(x))
    g = np.zeros_like(logits)
    for s, (a, b) in enumerate(zip(OFF, OFF[1:])):
        one = np.zeros((b - a, V))
        ok = target[a:b] >= 0
        one[np.nonzero(ok)[0], target[a:b][ok].astype(int)] = 1
        g[a:b] = (f[s // 2] if s % 2 == 0 else -f[s // 2]) * (one - soft[a:b]) * ok[:, None]
    return np.logaddexp(0, -x).mean(), g


def np_backward(m, g, ids):
    """Descent directions of every weight from that of the logits."""
    w, G = m["w"], H // HK
    dh = g @ w["emb"]
    demb = g.T @ m["hid"]
    dy, dqkv = dh @ w["proj"].T, np.zeros_like(m["qkv"])
    for s, (a, b) in enumerate(zip(OFF, OFF[1:])):
        for h in range(H):
            q, k, v = np_heads(m["qkv"][a:b], h)
            p, o = m["ps"][s, h], dy[a:b, h * D:(h + 1) * D]
            dp = o @ v.T
            ds = p * (dp - (dp * p).sum(1, keepdims=True)) * SCALE
            for at, d in ((h * D, ds @ k), ((H + h // G) * D, ds.T @ q), ((H + HK + h // G) * D, p.T @ o)):
                dqkv[a:b, at:at + D] += d
    dx = dqkv @ w["qkv"].T + dh
    np.add.at(demb, ids, dx)
    return dict(emb=demb, qkv=m["x"].T @ dqkv, proj=m["y"].T @ dh)


def test_numpy_gradients_against_differences():
    w, (ids, target) = weights(0), data()
    ref = np_logp(np_forward(weights(5), ids)["logits"], target)[1]
    _, g = np_loss(np_forward(w, ids)["logits"], target, ref, 0.3)
    grads = np_backward(np_forward(w, ids), g, ids)
    r = np.random.default_rng(2)
    for name in w:
        d = r.standard_normal(w[name].shape)
        loss = lambda t: np_loss(np_forward({**w, name: w[name].astype(np.float64) + t * d}, ids)["logits"], target, ref, 0.3)[0]  # noqa: E731,B023
        slope = (loss(1e-5) - loss(-1e-5)) / 2e-5
        assert abs(slope + np.sum(grads[name] * d)) <= 1e-6 * np.sum(np.abs(grads[name] * d)), name


# ---- the framework --------------------------------------------------------------------------------

class Model:
    def __init__(self, w, ids, target):
        dev, z = fh.DeviceArray.from_host, lambda *s: fh.DeviceArray.from_host(np.zeros(s, np.float32))  # noqa: E731
        self.w = {k: dev(x) for k, x in w.items()}
        self.g = {k: z(*x.shape) for k, x in w.items()}
        self.ids, self.target, self.off = dev(ids.astype(np.float32)), dev(target), dev(OFF)
        self.x, self.qkv, self.y, self.hid, self.logits = z(ROWS, C), z(ROWS, W), z(ROWS, H * D), z(ROWS, C), z(ROWS, V)
        self.lse, self.dh, self.dy, self.dqkv, self.dx = z(H, ROWS), z(ROWS, C), z(ROWS, H * D), z(ROWS, W), z(ROWS, C)
        self.loss, self.logp = z(1), z(len(LENS))
        self.shape = fh.PackedAttention(
            n_seq=len(LENS), q_rows=ROWS, k_rows=ROWS, n_head=H, n_kv_head=HK, head_dim=D, scale=SCALE, q_off=self.off.ptr,
            k_off=self.off.ptr, k_len=None, q_rs=W, o_rs=H * D, k_rs=W, v_rs=W, k_hs=D, v_hs=D)
        self.ws_n = max(1, fh.attention_packed_workspace(self.shape, True))
        self.ws, self.pws = z(self.ws_n), z(fh.preference_workspace(ROWS, len(LENS)))

    def attention(self, d):
        return d.ptr, d.at(H * D), d.at((H + HK) * D)

    def forward(self):
        fh.gather_rows(self.x.ptr, self.w["emb"].ptr, self.ids.ptr, C, ROWS, 1, V, 1)
        fh.mul(fh.NONE, self.qkv.ptr, self.x.ptr, self.w["qkv"].ptr, ROWS, W, C)
        fh.attention_packed(self.shape, self.y.ptr, self.lse.ptr, *self.attention(self.qkv), self.ws.ptr, self.ws_n)
        fh.gemm_ex(self.y.ptr, H * D, self.w["proj"].ptr, C, 0, self.hid.ptr, C, ROWS, C, H * D, fh.EPI_RESID, self.x.ptr, C)
        fh.mul(fh.RIGHT, self.logits.ptr, self.hid.ptr, self.w["emb"].ptr, ROWS, V, C)

    def logprobs(self):
        fh.sequence_logprobs(self.logp.ptr, self.pws.ptr, self.target.ptr, self.logits.ptr, self.off.ptr, V, ROWS, len(LENS))
        return self.logp.numpy()

    def backward(self, ref, beta):
        self.ref = fh.DeviceArray.from_host(ref)
        g = self.logits  # in place
        fh.preference_logits(g.ptr, self.loss.ptr, self.logp.ptr, self.pws.ptr, self.target.ptr, self.logits.ptr, self.off.ptr,
                             self.ref.ptr, V, ROWS, len(LENS) // 2, beta)
        fh.mul(fh.NONE, self.dh.ptr, g.ptr, self.w["emb"].ptr, ROWS, C, V)
        fh.mul(fh.LEFT, self.g["emb"].ptr, g.ptr, self.hid.ptr, V, C, ROWS)
        fh.mul(fh.LEFT, self.g["proj"].ptr, self.y.ptr, self.dh.ptr, H * D, C, ROWS)
        fh.mul(fh.RIGHT, self.dy.ptr, self.dh.ptr, self.w["proj"].ptr, ROWS, H * D, C)
        fh.attention_packed_backward(self.shape, *self.attention(self.dqkv), self.dy.ptr, self.y.ptr, self.lse.ptr,
                                     *self.attention(self.qkv), self.ws.ptr, self.ws_n)
        fh.mul(fh.LEFT, self.g["qkv"].ptr, self.x.ptr, self.dqkv.ptr, C, W, ROWS)
        fh.gemm_ex(self.dqkv.ptr, W, self.w["qkv"].ptr, W, 1, self.dx.ptr, C, ROWS, C, W, fh.EPI_RESID, self.dh.ptr, C)
        fh.scatter_add_rows(self.g["emb"].ptr, self.dx.ptr, self.ids.ptr, C, ROWS, 1, V, 1)


def far(got, ref):
    return np.linalg.norm(np.asarray(got, np.float64) - ref) / np.linalg.norm(ref)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_preference_step(bits):
    ids, target = data()
    w0, w = weights(5), weights(0)
    before = Model(w0, ids, target)
    before.forward()
    ref = before.logprobs()
    np_ref = np_logp(np_forward(w0, ids)["logits"], target)[1]
    assert far(ref, np_ref) < TOL

    m = Model(w, ids, target)
    m.forward()
    n = np_forward(w, ids)
    assert far(m.logits.numpy(), n["logits"]) < TOL
    m.backward(ref, 0.3)
    loss, g = np_loss(n["logits"], target, np_ref, 0.3)
    assert abs(m.loss.numpy()[0] / loss - 1) < TOL
    grads = np_backward(n, g, ids)
    for k in grads:
        assert far(m.g[k].numpy(), grads[k]) < TOL, k

    # One step from states of zero: every weight moves by the learning rate towards its gradient.
    names = list(w)
    blocks = {k: -(-w[k].size // 256) for k in names}
    dtype = np.float32 if bits == 32 else np.uint8
    st = {k: [fh.DeviceArray.from_host(np.zeros(s, t)) for s, t in ((w[k].size, dtype), (w[k].size, dtype), (blocks[k], np.uint8), (blocks[k], np.uint8))]
          for k in names}
    table = fh.adamw_tensors([(m.w[k].ptr, m.g[k].ptr, st[k][0].ptr, st[k][1].ptr, w[k].size) +
                              ((st[k][2].ptr, st[k][3].ptr) if bits == 8 else ()) for k in names])
    fh.adamw_update_multi(table, bits, LR, B1, B2, B1, B2, EPS, WD, 1)
    for k in names:
        gk = m.g[k].numpy().astype(np.float64)
        ref_w = w[k] + LR * gk / (np.abs(gk) + EPS) - LR * WD * w[k]
        assert np.max(np.abs(m.w[k].numpy() - ref_w)) <= 1e-6, k
    m.forward()  # the next forward pass takes the new weights
    new = {k: m.w[k].numpy() for k in names}
    assert far(m.logits.numpy(), np_forward(new, ids)["logits"]) < TOL

    # Serving: the longest sequence's keys and values in a cache, its last token as a single query.
    s, n_keys, T = 3, LENS[3], 64
    qkv = m.qkv.numpy()[OFF[s]:OFF[s + 1]]
    cache = np.zeros((2, HK, T, D), np.float32)
    for i in range(2):
        cache[i, :, :n_keys] = qkv[:, (H + i * HK) * D:(H + (i + 1) * HK) * D].reshape(n_keys, HK, D).transpose(1, 0, 2)
    dk, dv, dq = (fh.DeviceArray.from_host(x) for x in (cache[0], cache[1], qkv[-1:]))
    q_off, k_off, k_len = (fh.DeviceArray.from_host(np.array(x, np.int32)) for x in ([0, 1], [0, HK * T], [n_keys]))
    out = fh.DeviceArray((1, H * D))
    one = fh.PackedAttention(n_seq=1, q_rows=1, k_rows=HK * T, n_head=H, n_kv_head=HK, head_dim=D, scale=SCALE, q_off=q_off.ptr,
                             k_off=k_off.ptr, k_len=k_len.ptr, q_rs=W, o_rs=H * D, k_rs=D, v_rs=D, k_hs=T * D, v_hs=T * D)
    ws_n = fh.attention_packed_workspace(one)
    ws = fh.DeviceArray(max(1, ws_n))
    fh.attention_packed(one, out.ptr, 0, dq.ptr, dk.ptr, dv.ptr, ws.ptr, ws_n)
    assert far(out.numpy()[0], m.y.numpy()[OFF[s + 1] - 1]) < TOL
