"""Packed causal attention with grouped heads (fmlh_attention_packed and its backward) against the
formula in 64 bits.

Tolerances follow from the arithmetic, computed for each element from absolute values (u = 2^-24, half
a step of fp32 relative to the value).  A sum of n products in fp32 is off by at most n u times
the sum of their absolute values.  With A the largest scale * sum |q| |k| of a row and D dims, a score
is off by (D + 8) u A (product, scaling, the base-2 exponent's constant); a probability by ep =
2 (D + 8) u A + (n + 8) u relative (numerator, and its share in the sum of n; exp2 is within two units),
and out by sum p |v| (ep + n u).  A probability below 2^-126, fp32's smallest normal
number, may come out as zero (the hardware's exponential gives no subnormal ones): 2^-126 more, absolute.
lse, which the backward pass starts from, is off by (D + 8) u A + (n + 8) u and a rounding of its own size.  The gradients' bounds carry these on through their formulas.
"""
import numpy as np
import pytest

import freeml_amd as fh
from graphs import Captured

U = 2.0**-24
MARK = np.float32(123.25)  # what rows outside every sequence hold before and after


class Case:
    """Inputs of one call in host memory: packed QKV rows, slabs of a cache, or rows with odd strides
    and alignment; `extra` rows before and behind the sequences."""

    def __init__(self, qlens, klens, heads, kv_heads, dim, layout="qkv", extra=(0, 0), seed=0, scale=None, std=1.0):
        r = np.random.default_rng(seed)
        self.qlens, self.klens, self.H, self.Hk, self.D, self.layout = list(qlens), list(klens), heads, kv_heads, dim, layout
        self.n, self.scale = len(qlens), dim**-0.5 if scale is None else scale
        f = lambda *s: (std * r.standard_normal(s)).astype(np.float32)  # noqa: E731
        self.q = [f(n, heads, dim) for n in qlens]
        self.k = [f(n, kv_heads, dim) for n in klens]
        self.v = [f(n, kv_heads, dim) for n in klens]
        self.g = [f(n, heads, dim) for n in qlens]
        self.q_off = np.cumsum([extra[0]] + self.qlens).astype(np.int32)
        self.q_rows = int(self.q_off[-1]) + extra[1]
        H, Hk, D = heads, kv_heads, dim
        self.k_len = None
        if layout == "qkv":
            assert self.qlens == self.klens
            self.shift, w = 0, (H + 2 * Hk) * D
            self.k_off, self.k_rows = self.q_off, self.q_rows
            self.q_rs = self.k_rs = self.v_rs = w
            self.o_rs, self.k_hs, self.v_hs = H * D, D, D
        elif layout == "cache":
            T = max(self.klens) + 3
            self.shift = 0
            self.k_off = (np.arange(self.n + 1) * Hk * T).astype(np.int32)
            self.k_len = np.array(self.klens, np.int32)
            self.k_rows = self.n * Hk * T
            self.q_rs, self.o_rs, self.k_rs, self.v_rs, self.k_hs, self.v_hs = (H + 1) * D, H * D, D, D, T * D, T * D
        else:  # odd strides, 4-byte alignment
            self.shift = 1
            self.k_off = np.cumsum([extra[0]] + self.klens).astype(np.int32)
            self.k_rows = int(self.k_off[-1]) + extra[1]
            self.q_rs, self.o_rs = H * D + 3, H * D + 1
            self.k_hs, self.v_hs = D + 5, D + 2
            self.k_rs, self.v_rs = Hk * self.k_hs + 7, Hk * self.v_hs

    def _buffer(self, n):
        return np.full(self.shift + n + 8, MARK, np.float32)

    def _view(self, buf, rows, rs, heads, hs, at=0):
        s = buf[self.shift + at:]
        return np.lib.stride_tricks.as_strided(s, (rows, heads, self.D), (4 * rs, 4 * hs, 4), writeable=True)

    def _key_view(self, buf, s, rs, hs, at=0):
        return self._view(buf, self.klens[s], rs, self.Hk, hs, at + int(self.k_off[s]) * rs)

    def build(self):
        """Device arrays and the views' places."""
        H, Hk, D = self.H, self.Hk, self.D
        self.places = {}
        if self.layout == "qkv":
            buf = self._buffer(self.q_rows * self.q_rs)
            self.places = dict(q=(0, 0), k=(0, H * D), v=(0, (H + Hk) * D))
            bufs = [buf]
        else:
            bufs = [self._buffer(self.q_rows * self.q_rs), self._buffer(self.k_rows * self.k_rs + Hk * self.k_hs),
                    self._buffer(self.k_rows * self.v_rs + Hk * self.v_hs)]
            self.places = dict(q=(0, 0), k=(1, 0), v=(2, 0))
        self.blank = [b.copy() for b in bufs]
        for s in range(self.n):
            if self.qlens[s]:
                i, at = self.places["q"]
                self._view(bufs[i], self.qlens[s], self.q_rs, H, D, at + int(self.q_off[s]) * self.q_rs)[:] = self.q[s]
            if self.klens[s]:
                for name, x, rs, hs in (("k", self.k, self.k_rs, self.k_hs), ("v", self.v, self.v_rs, self.v_hs)):
                    i, at = self.places[name]
                    self._key_view(bufs[i], s, rs, hs, at)[:] = x[s]
        rows = self._buffer(self.q_rows * self.o_rs)
        self.out_blank = rows.copy()
        for s in range(self.n):
            if self.qlens[s]:
                self._view(rows, self.qlens[s], self.o_rs, H, D, int(self.q_off[s]) * self.o_rs)[:] = self.g[s]
        dev = fh.DeviceArray.from_host
        self.d_in, self.d_g = [dev(b) for b in bufs], dev(rows)
        self.d_out, self.d_lse = dev(self.out_blank), dev(np.full((H, self.q_rows), MARK, np.float32))
        self.d_grad = [dev(b) for b in self.blank]
        self.d_off = [dev(self.q_off), dev(self.k_off)] + ([dev(self.k_len)] if self.k_len is not None else [])
        self.shape = fh.PackedAttention(
            n_seq=self.n, q_rows=self.q_rows, k_rows=self.k_rows, n_head=H, n_kv_head=Hk, head_dim=D, scale=self.scale,
            q_off=self.d_off[0].ptr, k_off=self.d_off[1].ptr, k_len=self.d_off[2].ptr if self.k_len is not None else None,
            q_rs=self.q_rs, o_rs=self.o_rs, k_rs=self.k_rs, v_rs=self.v_rs, k_hs=self.k_hs, v_hs=self.v_hs)
        n = max(fh.attention_packed_workspace(self.shape), fh.attention_packed_workspace(self.shape, True), 1)
        self.d_ws, self.ws_n = dev(np.full(n, np.nan, np.float32)), n
        return self

    def at(self, arrays, name):
        i, at = self.places[name]
        return arrays[i].at(self.shift + at)

    def forward(self, lse=True):
        fh.attention_packed(self.shape, self.d_out.at(self.shift), self.d_lse.ptr if lse else 0,
                            *(self.at(self.d_in, x) for x in "qkv"), self.d_ws.ptr, self.ws_n)

    def backward(self):
        fh.attention_packed_backward(self.shape, *(self.at(self.d_grad, x) for x in "qkv"), self.d_g.at(self.shift),
                                     self.d_out.at(self.shift), self.d_lse.ptr, *(self.at(self.d_in, x) for x in "qkv"),
                                     self.d_ws.ptr, self.ws_n)

    def read_rows(self, buf):
        return [self._view(buf, n, self.o_rs, self.H, self.D, int(o) * self.o_rs).copy() if n else np.zeros((0, self.H, self.D), np.float32)
                for n, o in zip(self.qlens, self.q_off)]

    def read_grads(self):
        bufs = [d.numpy() for d in self.d_grad]
        got, (i, at) = {}, self.places["q"]
        got["q"] = [self._view(bufs[i], n, self.q_rs, self.H, self.D, at + int(o) * self.q_rs).copy() if n else np.zeros((0, self.H, self.D))
                    for n, o in zip(self.qlens, self.q_off)]
        for name, rs, hs in (("k", self.k_rs, self.k_hs), ("v", self.v_rs, self.v_hs)):
            i, at = self.places[name]
            got[name] = [self._key_view(bufs[i], s, rs, hs, at).copy() if self.klens[s] else np.zeros((0, self.Hk, self.D))
                         for s in range(self.n)]
        return got, bufs

    def untouched(self, bufs, which):
        """No byte outside the sequences' rows changed."""
        if which == "out":
            b = bufs.copy()
            for s in range(self.n):
                if self.qlens[s]:
                    self._view(b, self.qlens[s], self.o_rs, self.H, self.D, int(self.q_off[s]) * self.o_rs)[:] = MARK
            assert np.all(b == MARK)
            return
        bufs = [b.copy() for b in bufs]
        for s in range(self.n):
            if self.qlens[s]:
                i, at = self.places["q"]
                self._view(bufs[i], self.qlens[s], self.q_rs, self.H, self.D, at + int(self.q_off[s]) * self.q_rs)[:] = MARK
            if self.klens[s]:
                for name, rs, hs in (("k", self.k_rs, self.k_hs), ("v", self.v_rs, self.v_hs)):
                    i, at = self.places[name]
                    self._key_view(bufs[i], s, rs, hs, at)[:] = MARK
        assert all(np.all(b == MARK) for b in bufs)


def reference(c, s, h, k=None, v=None):
    """Of sequence s and head h in 64 bits: out, lse, gradients and the bound of every one of them."""
    G, D = c.H // c.Hk, c.D
    q, g = c.q[s][:, h].astype(np.float64), c.g[s][:, h].astype(np.float64)
    k = (c.k if k is None else k)[s][:, h // G].astype(np.float64)
    v = (c.v if v is None else v)[s][:, h // G].astype(np.float64)
    ql, kl = len(q), len(k)
    scale = float(np.float32(c.scale))
    seen = np.arange(kl) <= np.arange(ql)[:, None] + kl - ql
    x = np.where(seen, q @ k.T * scale, -np.inf)
    top = np.max(x, axis=1, keepdims=True, initial=-np.inf)
    top = np.where(np.isfinite(top), top, 0.0)
    e = np.exp(x - top)
    total = e.sum(1, keepdims=True)
    p = e / np.where(total == 0, 1.0, total)
    with np.errstate(divide="ignore"):
        lse = (top + np.log(total))[:, 0]
    out = p @ v
    A = np.max(np.where(seen, np.abs(q) @ np.abs(k).T * abs(scale), 0.0), axis=1, keepdims=True, initial=0.0)
    n = kl + 8
    ep = 2 * (D + 8) * U * A + n * U
    fin = np.where(np.isfinite(lse), np.abs(lse), 0.0)
    low = np.where(seen, 2.0**-126, 0.0)  # of a probability that came out as zero
    b_out = p @ np.abs(v) * (ep + n * U) + low @ np.abs(v)
    b_lse = ((D + 8) * U * A + n * U)[:, 0] + 2 * U * fin
    ep = ep + b_lse[:, None] + 4 * U * fin[:, None]  # p again, from lse
    dp, absdp = g @ v.T, np.abs(g) @ np.abs(v).T
    d, absd = (g * out).sum(1, keepdims=True), (np.abs(g) * np.abs(out)).sum(1, keepdims=True)
    ds = p * (dp - d) * scale
    b_ds = abs(scale) * p * (np.abs(dp - d) * (ep + 4 * U) + (absdp + absd) * (D + 8) * U + (np.abs(g) * b_out).sum(1, keepdims=True))
    b_ds += abs(scale) * low * np.abs(dp - d)
    m = ql * G + 8
    return dict(out=out, lse=lse, q=ds @ k, k=ds.T @ q, v=p.T @ g, b_out=b_out, b_lse=b_lse,
                b_q=b_ds @ np.abs(k) + np.abs(ds) @ np.abs(k) * n * U, b_k=b_ds.T @ np.abs(q) + np.abs(ds).T @ np.abs(q) * m * U,
                b_v=(p * ep + low).T @ np.abs(g) + p.T @ np.abs(g) * m * U)


def close(got, ref, bound, what):
    got = np.asarray(got, np.float64)
    assert got.shape == ref.shape
    with np.errstate(invalid="ignore"):
        far = np.abs(got - ref) - bound - np.abs(ref) * U - 2.0**-126
    ok = (far <= 0) | (got == ref)
    assert np.all(ok), f"{what}: {np.sum(~ok)} of {ok.size} off, worst {np.nanmax(np.abs(got - ref) / (bound + 1e-300)):.3g} bounds"


def check(c, backward=True):
    c.build()
    c.forward()
    buf, lse = c.d_out.numpy(), c.d_lse.numpy()
    c.untouched(buf, "out")
    outs = c.read_rows(buf)
    if backward:
        c.backward()
        grads, bufs = c.read_grads()
        c.untouched(bufs, "grad")
    G = c.H // c.Hk
    in_seq = np.zeros(c.q_rows, bool)
    for s in range(c.n):
        rows = slice(int(c.q_off[s]), int(c.q_off[s]) + c.qlens[s])
        in_seq[rows] = True
        for hk in range(c.Hk):
            refs = [reference(c, s, h) for h in range(hk * G, (hk + 1) * G)]
            for i, h in enumerate(range(hk * G, (hk + 1) * G)):
                r = refs[i]
                close(outs[s][:, h], r["out"], r["b_out"], f"out of sequence {s}, head {h}")
                close(lse[h, rows], r["lse"], r["b_lse"], f"lse of sequence {s}, head {h}")
                if backward:
                    close(grads["q"][s][:, h], r["q"], r["b_q"], f"dq of sequence {s}, head {h}")
            if backward:
                for x in "kv":
                    close(grads[x][s][:, hk], sum(r[x] for r in refs), sum(r["b_" + x] for r in refs), f"d{x} of sequence {s}, key head {hk}")
    assert np.all(lse[:, ~in_seq] == MARK)


WHOLE = [
    ([1], 1, 1, 64), ([5], 2, 1, 16), ([33, 1, 64], 4, 4, 64), ([130, 7], 6, 2, 64), ([65], 3, 3, 32), ([40, 129], 4, 1, 128),
    ([100], 8, 2, 80), ([31, 32], 2, 2, 1), ([50], 2, 1, 37), ([257, 300], 2, 2, 96), ([0, 9, 0, 3], 2, 1, 64), ([700], 1, 1, 64),
    ([64, 128, 191], 5, 1, 128), ([1, 1, 1, 2], 12, 4, 64),
]


@pytest.mark.gpu
@pytest.mark.parametrize("lens,heads,kv_heads,dim", WHOLE)
def test_whole_sequences(lens, heads, kv_heads, dim):
    print(f"whole sequences {lens} heads {heads}/{kv_heads} of {dim}", flush=True)
    check(Case(lens, lens, heads, kv_heads, dim, extra=(2, 3), seed=sum(lens) + dim))


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["cache", "odd"])
@pytest.mark.parametrize("qlens,klens,heads,kv_heads,dim", [
    ([1] * 5, [1, 2, 33, 300, 64], 4, 4, 64), ([1, 1], [700, 1500], 8, 2, 128), ([3, 48], [500, 50], 4, 2, 80), ([7, 1, 0], [7, 90, 20], 2, 1, 64),
    ([1], [5000], 2, 1, 64), ([20, 130], [5, 140], 2, 2, 32), ([4], [0], 2, 1, 64), ([1] * 70, list(range(1, 71)), 2, 1, 16),
    ([1], [129], 1, 1, 33)])
def test_queries_over_longer_keys(layout, qlens, klens, heads, kv_heads, dim):
    """Single tokens and chunks over a cache; more queries than keys leave the first rows empty."""
    print(f"{layout} queries {qlens[:5]} keys {klens[:5]} heads {heads}/{kv_heads} of {dim}", flush=True)
    check(Case(qlens, klens, heads, kv_heads, dim, layout, extra=(1, 2) if layout == "odd" else (0, 0), seed=len(qlens) + dim))


@pytest.mark.gpu
@pytest.mark.parametrize("lens,heads,kv_heads,dim", [([1700], 2, 1, 64), ([1600, 1550], 1, 1, 33), ([2100], 1, 1, 24), ([900, 1300], 2, 2, 128)])
def test_long_sequences(lens, heads, kv_heads, dim):
    """From 1536 keys on four pairs of waves share a tile of the backward pass; few tiles of long keys are cut."""
    check(Case(lens, lens, heads, kv_heads, dim, extra=(1, 0), seed=dim))


@pytest.mark.gpu
def test_more_work_than_runs_at_once():
    """Up to 64 sequences in the order of their work: every tile once, whatever the lengths."""
    r = np.random.default_rng(5)
    lens = r.integers(0, 400, 60).tolist()
    check(Case(lens, lens, 6, 6, 16, seed=11))


@pytest.mark.gpu
@pytest.mark.parametrize("qlens", [[1, 1, 1], [3, 2, 2], [200, 70, 300]])
def test_caches_without_a_key(qlens):
    """Room for many keys, none of them written: every row is there and empty."""
    c = Case(qlens, [900, 800, 700], 4, 2, 64, "cache").build()
    c.klens = [0, 0, 0]
    c.d_off[2].upload(np.zeros(3, np.int32))
    c.forward()
    out, lse = c.d_out.numpy(), c.d_lse.numpy()
    assert all(np.all(x == 0.0) for x in c.read_rows(out)) and np.all(lse == -np.inf)
    c.untouched(out, "out")


@pytest.mark.gpu
def test_many_sequences():
    r = np.random.default_rng(4)
    lens = r.integers(0, 12, 300).tolist()
    check(Case(lens, lens, 2, 1, 32, seed=9))


@pytest.mark.gpu
@pytest.mark.parametrize("std", [1e-12, 30.0, 1e4])
def test_sizes_of_values(std):
    """Scores near zero (an even softmax) and in the thousands (one key takes all)."""
    check(Case([90, 40], [90, 40], 4, 2, 64, seed=5, std=std, scale=0.125 if std < 1e3 else 1e-6))


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("v,g", [(1e30, 1.0), (1e-30, 1e30), (1.0, 1e-34), (1e-34, 1.0), (1e34, 1e-34), (1e-20, 1e-12)])
def test_values_and_gradients_at_the_ends_of_the_range(v, g, dim):
    """Operands whose parts or sums leave the range of the bf16 products, at either end, lose nothing."""
    c = Case([70, 33], [70, 33], 4, 2, dim, seed=13)
    c.v = [(x * np.float32(v)).astype(np.float32) for x in c.v]
    c.g = [(x * np.float32(g)).astype(np.float32) for x in c.g]
    check(c)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [20, 64, 128])
@pytest.mark.parametrize("v", [1.0, 1e30])
@pytest.mark.parametrize("heads", [4, 96])
def test_tiles_of_all_and_of_half_the_rows(heads, v, dim):
    """Few tiles take half the rows each, many (96 heads) all of them; lengths at and around both."""
    lens = [63, 64, 65, 1, 128, 129, 32, 97] if heads == 4 else [130, 66, 1]
    c = Case(lens, lens, heads, heads // 2, dim, seed=21)
    c.v = [(x * np.float32(v)).astype(np.float32) for x in c.v]
    check(c)


@pytest.mark.gpu
def test_bad_keys_behind_a_row_in_the_same_tile():
    """Half-row tiles whose second waves hold nothing but masked keys, some of them not finite."""
    c = Case([40], [40], 2, 2, 32, seed=22)
    clean = Case([40], [40], 2, 2, 32, seed=22)
    c.k[0][33:] = np.nan
    c.v[0][33:] = np.inf
    c.build()
    c.forward()
    out, lse = c.read_rows(c.d_out.numpy()), c.d_lse.numpy()
    for h in range(2):
        r = reference(clean, 0, h)
        close(out[0][:33, h], r["out"][:33], r["b_out"][:33], "out")
        close(lse[h, :33], r["lse"][:33], r["b_lse"][:33], "lse")


@pytest.mark.gpu
@pytest.mark.parametrize("klens", [[3000], [900, 2000]])
def test_cut_keys_at_the_ends_of_the_range(klens):
    """The same where the keys are cut into ranges, on tiles of rows and on few rows."""
    for n in (40, 1):
        c = Case([n] * len(klens), klens, 4, 2, 64, "cache", seed=14)
        c.v = [x * np.float32(1e30) for x in c.v]
        check(c, backward=False)


@pytest.mark.gpu
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("dim", [64, 128])
def test_masked_places_may_hold_anything(value, dim):
    """Values that are not finite in the rows of position 70 on reach neither the rows before it
    nor any other sequence; rows from 70 on are not finite."""
    c = Case([100, 60], [100, 60], 4, 2, dim, seed=6)
    clean = Case([100, 60], [100, 60], 4, 2, dim, seed=6)
    for x in (c.q, c.k, c.v, c.g):
        x[0][70:] = value
    c.build()
    c.forward()
    c.backward()
    outs, lse = c.read_rows(c.d_out.numpy()), c.d_lse.numpy()
    grads, _ = c.read_grads()
    for h in range(4):
        for s, n in ((0, 70), (1, 60)):
            r = reference(clean, s, h)
            close(outs[s][:n, h], r["out"][:n], r["b_out"][:n], "out")
            close(lse[h, c.q_off[s]:c.q_off[s] + n], r["lse"][:n], r["b_lse"][:n], "lse")
            close(grads["q"][s][:n, h], r["q"][:n], r["b_q"][:n], "dq")
        assert not np.any(np.isfinite(outs[0][70:, h]))
    for hk in range(2):
        for x in "kv":
            refs = [reference(clean, 1, h) for h in (2 * hk, 2 * hk + 1)]
            close(grads[x][1][:, hk], sum(r[x] for r in refs), sum(r["b_" + x] for r in refs), "d" + x)


@pytest.mark.gpu
def test_gradient_of_rows_that_follow_a_bad_query():
    """A query whose gradient is not finite leaves the keys behind it alone."""
    c = Case([96], [96], 2, 1, 64, seed=8)
    clean = Case([96], [96], 2, 1, 64, seed=8)
    c.g[0][:40] = np.inf
    clean.g[0][:40] = 0.0
    c.build()
    c.forward()
    c.backward()
    grads, _ = c.read_grads()
    refs = [reference(clean, 0, h) for h in range(2)]
    for x in "kv":
        close(grads[x][0][40:, 0], sum(r[x] for r in refs)[40:], sum(r["b_" + x] for r in refs)[40:], "d" + x)


@pytest.mark.gpu
def test_scores_of_minus_infinity_count_as_nothing():
    c = Case([40], [40], 1, 1, 32, seed=3)
    c.q[0][:, 0, 0] = np.abs(c.q[0][:, 0, 0]) + 1
    c.k[0][1::3, 0, 0] = -np.inf
    c.build()
    c.forward()
    with np.errstate(invalid="ignore"):
        x = c.q[0][:, 0].astype(np.float64) @ c.k[0][:, 0].astype(np.float64).T * c.scale
    x[np.arange(40) > np.arange(40)[:, None]] = -np.inf
    p = np.exp(x - x.max(1, keepdims=True))
    ref = p / p.sum(1, keepdims=True) @ c.v[0][:, 0].astype(np.float64)
    np.testing.assert_allclose(c.read_rows(c.d_out.numpy())[0][:, 0], ref, atol=1e-5)


@pytest.mark.gpu
def test_gradients_against_differences():
    """Central differences of sum(out dout) along random directions.  With steps of 2^-7 the second-order
    term is below 1e-3 of the derivative's size here; rounding of out adds 2^-24 sum |out dout| / 2^-7."""
    r = np.random.default_rng(12)
    c = Case([50, 20], [50, 20], 4, 2, 64, seed=12).build()
    c.forward()
    c.backward()
    grads, _ = c.read_grads()

    def total(step, direction, name):
        d = Case([50, 20], [50, 20], 4, 2, 64, seed=12)
        for s in range(2):
            getattr(d, name)[s] = (getattr(d, name)[s] + np.float32(step) * direction[s]).astype(np.float32)
        d.build()
        d.forward(lse=False)
        return sum(np.sum(o.astype(np.float64) * g) for o, g in zip(d.read_rows(d.d_out.numpy()), d.g))

    for name in "qkv":
        direction = [r.choice([-1.0, 1.0], x.shape).astype(np.float32) for x in getattr(c, name)]
        diff = (total(2.0**-7, direction, name) - total(-(2.0**-7), direction, name)) * 2.0**6
        exact = sum(np.sum(a.astype(np.float64) * b) for a, b in zip(grads[name], direction))
        size = sum(np.sum(np.abs(a)) for a in grads[name])
        assert abs(diff - exact) <= 2e-3 * size, (name, diff, exact, size)


@pytest.mark.gpu
def test_same_bits_every_time_and_on_other_workspaces():
    c = Case([200, 30, 1], [200, 30, 1], 8, 2, 64, seed=2).build()
    seen = []
    for _ in range(3):
        c.forward()
        c.backward()
        seen.append([c.d_out.numpy(), c.d_lse.numpy()] + [d.numpy() for d in c.d_grad])
        c.d_ws.upload(np.full(c.ws_n, 7.0, np.float32))
    for other in seen[1:]:
        for a, b in zip(seen[0], other):
            np.testing.assert_array_equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("stride", [1 << 22, (1 << 22) + 4])
def test_wide_row_strides(stride):
    """Keys far apart, up to and beyond the stride that vector loads take: the bits of close ones."""
    r, n, H, D = np.random.default_rng(31), 5, 2, 64
    dev = fh.DeviceArray.from_host
    off = dev(np.array([0, n], np.int32))
    q = dev(r.standard_normal((n, H * D)).astype(np.float32))
    kv = r.standard_normal((n, 2 * H * D)).astype(np.float32)
    wide = np.zeros((n, stride), np.float32)
    wide[:, :2 * H * D] = kv
    results = []
    for keys, rs in ((kv, 2 * H * D), (wide, stride)):
        d_kv, out, lse = dev(keys), dev(np.zeros((n, H * D), np.float32)), dev(np.zeros((H, n), np.float32))
        shape = fh.PackedAttention(n_seq=1, q_rows=n, k_rows=n, n_head=H, n_kv_head=1, head_dim=D, scale=0.125, q_off=off.ptr,
                                   k_off=off.ptr, k_len=None, q_rs=H * D, o_rs=H * D, k_rs=rs, v_rs=rs, k_hs=D, v_hs=D)
        assert fh.attention_packed_workspace(shape) == 0
        fh.attention_packed(shape, out.ptr, lse.ptr, q.ptr, d_kv.ptr, d_kv.at(H * D))
        results.append((out.numpy(), lse.numpy()))
    assert np.all(results[0][0] == results[1][0]) and np.all(results[0][1] == results[1][1])
    assert np.any(results[0][0] != 0)


@pytest.mark.gpu
def test_offsets_outside_the_rows_are_cut():
    """Offsets beyond the rows that exist, negative ones and lengths below zero read and write nothing outside."""
    c = Case([10, 20], [10, 20], 2, 1, 64, seed=1).build()
    c.d_off[0].upload(np.array([-5, 10, 4000], np.int32))
    c.forward()
    c.backward()
    outs = c.read_rows(c.d_out.numpy())
    r = reference(c, 0, 0)
    close(outs[0][:, 0], r["out"], r["b_out"], "out")
    r = reference(c, 1, 1)
    close(outs[1][:, 1], r["out"], r["b_out"], "out")
    d = Case([1, 1], [5, 6], 2, 1, 64, "cache", seed=1).build()
    d.d_off[2].upload(np.array([-3, 6], np.int32))
    d.forward()
    outs = d.read_rows(d.d_out.numpy())
    assert np.all(outs[0] == 0)
    r = reference(d, 1, 0)
    close(outs[1][:, 0], r["out"], r["b_out"], "out")


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [([60, 5], [60, 5], 4, 2, 64, "qkv"), ([1] * 4, [900, 3, 77, 400], 8, 2, 64, "cache")])
def test_captured_and_replayed(shape):
    """Replays follow the data and the lengths, with eager calls of the same buffers between them."""
    c = Case(*shape[:5], shape[5], seed=20).build()

    def calls():
        c.forward()
        c.backward()

    calls()
    g = Captured(calls)
    r = np.random.default_rng(0)
    for n in range(4):
        new = [np.where(b == MARK, b, r.standard_normal(b.shape).astype(np.float32)) for b in [d.numpy() for d in c.d_in]]
        for d, b in zip(c.d_in, new):
            d.upload(b)
        if c.k_len is not None:
            c.d_off[2].upload(np.maximum(1, c.k_len - n).astype(np.int32))
        got = []
        for replay in (False, True):
            for d, b in zip([c.d_out] + c.d_grad, [c.out_blank] + c.blank):
                d.upload(b)
            if replay:
                g.replay()
            else:
                calls()
            got.append([c.d_out.numpy(), c.d_lse.numpy()] + [d.numpy() for d in c.d_grad])
        for a, b in zip(*got):
            np.testing.assert_array_equal(a, b)


@pytest.mark.gpu
def test_forward_and_backward_follow_the_per_head_operators():
    """One sequence, as many key heads as heads: the score-matrix operators give the same."""
    T, H, D = 48, 3, 32
    c = Case([T], [T], H, H, D, seed=30).build()
    c.forward()
    out = c.read_rows(c.d_out.numpy())[0]
    scores = np.stack([c.q[0][:, h] @ c.k[0][:, h].T for h in range(H)]).astype(np.float32)
    dS, dP = fh.DeviceArray.from_host(scores), fh.DeviceArray((H, T, T))
    heads = [fh.DeviceArray((T, T)) for _ in range(H)]
    scale = fh.DeviceArray.from_host(np.array([c.scale], np.float32))
    fh.attention_softmax_heads([p.ptr for p in heads], 0, dP.ptr, dS.ptr, scale.ptr, H, T)
    p = dP.numpy()
    for h in range(H):
        np.testing.assert_allclose(out[:, h], p[h].astype(np.float64) @ c.v[0][:, h], atol=2e-5)


# ---- refusals (no device needed) -----------------------------------------------------------------

def shape(**over):
    f = dict(n_seq=1, q_rows=4, k_rows=4, n_head=4, n_kv_head=2, head_dim=8, scale=0.3, q_off=4096, k_off=4096, k_len=None,
             q_rs=32, o_rs=32, k_rs=16, v_rs=16, k_hs=8, v_hs=8)
    f.update(over)
    return fh.PackedAttention(**f)


BAD = [dict(n_head=0), dict(n_kv_head=0), dict(n_head=5), dict(head_dim=0), dict(head_dim=129), dict(q_off=None), dict(k_off=None),
       dict(q_rs=31), dict(o_rs=8), dict(k_rs=7), dict(v_rs=7), dict(k_hs=7), dict(v_hs=1), dict(scale=float("nan")),
       dict(scale=float("inf")), dict(scale=1e-19), dict(scale=-1e19), dict(q_rows=2**30 + 1), dict(k_rows=2**31), dict(n_seq=2**22 + 1), dict(q_rows=2**30, n_kv_head=1),
       dict(q_rs=2**32), dict(n_head=65536, n_kv_head=65536, q_rs=2**20, o_rs=2**20)]


@pytest.mark.parametrize("over", BAD, ids=[next(iter(b)) + str(i) for i, b in enumerate(BAD)])
def test_refused_shapes(over):
    a = shape(**over)
    for f in (lambda: fh.attention_packed_workspace(a), lambda: fh.attention_packed(a, 16, 16, 16, 16, 16, 16, 1 << 30),
              lambda: fh.attention_packed_backward(a, *[16] * 9, 16, 1 << 30)):
        with pytest.raises(fh.FreeMLHipError) as e:
            f()
        assert e.value.code == -1


def test_refused_pointers_and_workspaces():
    a = shape()
    for args in ([0, 16, 16, 16, 16], [16, 16, 0, 16, 16], [16, 16, 16, 0, 16], [16, 16, 16, 16, 0]):
        with pytest.raises(fh.FreeMLHipError) as e:
            fh.attention_packed(a, *args)
        assert e.value.code == -1
    for i in range(9):
        with pytest.raises(fh.FreeMLHipError) as e:
            fh.attention_packed_backward(a, *[0 if j == i else 16 for j in range(9)], 16, 1 << 20)
        assert e.value.code == -1
    with pytest.raises(fh.FreeMLHipError):
        fh.call("fmlh_attention_packed", None, 16, 16, 16, 16, 16, 16, 1)


def test_nothing_to_do_needs_nothing():
    fh.attention_packed(shape(n_seq=0, q_off=None, k_off=None), 0, 0, 0, 0, 0)
    fh.attention_packed(shape(q_rows=0), 0, 0, 0, 0, 0)
    fh.attention_packed_backward(shape(q_rows=0, k_rows=0), *[0] * 9)
