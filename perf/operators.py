"""Operators of preference tuning and of serving with grouped heads, as cases that can be timed and
checked.

* ``attend``: causal attention of packed sequences of different lengths, forward only: whole prompts
  out of the packed QKV rows, or a few new tokens of every sequence over a key/value cache.
* ``attend_train``: the same on whole sequences, forward and backward, into a packed QKV gradient.
* ``prefer``: the preference loss (paired log ratios) on logits and its gradient; ``logprobs``: the
  sequences' log-probabilities alone, as a reference model is asked for them.
* ``adamw``: one AdamW step over all tensors of a model, states in 32 or in 8 bits.  It changes
  parameters and states in place, as a training step does.

``own`` false: elementary torch operations in 32 bits (64 for the sums of log-probabilities).
Everything a user holds is fp32 but the 8-bit states.
"""
import math
import random

import torch

own = False

BLOCK = 256  # elements that share the scale of an 8-bit state


def _attend(name, kind, seqs, lo, hi, heads, kv_heads, dim, new=0, cache=0, mix=1):
    """new = 0: whole sequences of lo .. hi rows; else `new` rows each over lo .. hi keys, kept in
    slabs of `cache` positions per sequence and head (0: packed rows)."""
    c = dict(kind=kind, seqs=seqs, lo=lo, hi=hi, heads=heads, kv_heads=kv_heads, dim=dim, new=new, cache=cache, mix=mix)
    return dict(c, name=name) if name else c


def _prefer(name, kind, pairs, lo, hi, vocab, mix=1, smoothing=0.0):
    c = dict(kind=kind, pairs=pairs, lo=lo, hi=hi, vocab=vocab, mix=mix, smoothing=smoothing)
    return dict(c, name=name) if name else c


def _adamw(name, bits, vocab, block, embed, layers, step):
    c = dict(kind="adamw", bits=bits, vocab=vocab, block=block, embed=embed, layers=layers, step=step)
    return dict(c, name=name) if name else c


def listed():
    return [
        # 64 users of a character GPT, one token each over caches of up to 256 positions: latency.
        _attend("decode_64_users", "attend", 64, 64, 256, 6, 6, 64, new=1, cache=256),
        # Long conversations, one token each, four query heads on a key head: the cache's bytes.
        _attend("decode_long_grouped", "attend", 8, 2048, 32768, 32, 8, 128, new=1, cache=32768),
        # A chunk of 48 new tokens for each of four conversations, heads of 80.
        _attend("extend_chunk", "attend", 4, 500, 4000, 16, 4, 80, new=48, cache=4096),
        # Prompts of uneven length for a context of 4096.
        _attend("prompts_uneven", "attend", 6, 1000, 3584, 8, 8, 64),
        # A training batch of a character GPT: short sequences packed into one matrix.
        _attend("train_short", "attend_train", 16, 20, 256, 6, 6, 64),
        # Preference pairs packed at GPT-2-small's width, three query heads on a key head.
        _attend("train_packed_grouped", "attend_train", 24, 100, 2048, 12, 4, 64),
        # Two long sequences, heads of 128, eight query heads on a key head.
        _attend("train_long_128", "attend_train", 2, 3000, 4096, 16, 2, 128),
        # Preference tuning of a character GPT: many short rows.
        _prefer("prefer_char", "prefer", 32, 20, 256, 65),
        # Preference tuning with a vocabulary of 50304: the logits' bytes.
        _prefer("prefer_50304", "prefer", 6, 64, 640, 50304, smoothing=0.1),
        # The reference model's answers of the same pairs, vocabulary of an odd size.
        _prefer("logprobs_odd", "logprobs", 8, 32, 512, 32003),
        # The optimiser's step of a character GPT: 40 tensors from 384 to 590k elements.
        _adamw("adamw_32", 32, 65, 256, 384, 6, 1000),
        # The optimiser's step at GPT-2-small's size, states in 8 bits.
        _adamw("adamw_8", 8, 50304, 1024, 768, 12, 1000),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "attend_train", "attend_train", "prefer", "logprobs", "adamw"])
    while True:
        mix = rng.randint(2, 10**6)
        if kind in ("attend", "attend_train"):
            kv_heads = rng.choice([1, 2, 3, 4, 6, 8, 12])
            heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 8])
            dim = rng.choice([16, 32, 40, 64, 64, 64, 80, 96, 128, 128])
            seqs = _log_int(rng, 1, 64)
            hi = _log_int(rng, 1, 32768 if kind == "attend" else 4096)
            lo = _log_int(rng, 1, hi)
            new = rng.choice([0, 1, 1, 2, 5, 31, 130]) if kind == "attend" else 0
            cache = hi + rng.randint(0, 64) if new and rng.random() < 0.7 else 0
            c = _attend(None, kind, seqs, lo, hi, heads, kv_heads, dim, new, cache, mix)
            w = work(c)
            padded = seqs * heads * hi * (new or hi)  # scores of the plain form
            slabs = seqs * kv_heads * max(cache, hi) * dim
            if heads <= 32 and w["flops"] <= 4e11 and w["bytes"] <= 1.2e9 and padded <= 6e8 and slabs <= 5e8:
                return c
        elif kind in ("prefer", "logprobs"):
            hi = _log_int(rng, 1, 1024)
            c = _prefer(None, kind, _log_int(rng, 1, 64), _log_int(rng, 1, hi), hi, _log_int(rng, 33, 50304), mix,
                        rng.choice([0.0, 0.0, 0.1]))
            if sum(_lengths(c)) * c["vocab"] <= 1.3e8:
                return c
        else:
            c = _adamw(None, rng.choice([8, 32]), _log_int(rng, 33, 50304), _log_int(rng, 33, 2048), 8 * _log_int(rng, 2, 96),
                       rng.randint(1, 12), rng.randint(1, 100000))
            if sum(_sizes(c)) <= 1.2e8:
                return c


# ---- sizes -------------------------------------------------------------------------------------

def _lengths(case):
    """The sequences' lengths, a fixed function of the case."""
    r = random.Random(case["mix"])
    n = case["seqs"] if "seqs" in case else 2 * case["pairs"]
    return [_log_int(r, case["lo"], case["hi"]) for _ in range(n)]


def _query_lengths(case, lens):
    return [min(case["new"], k) for k in lens] if case["new"] else lens


def _sizes(case):
    """Elements of a NanoLLM's parameters: embeddings, the layers' four projections and two gains, the last gain."""
    V, T, C = case["vocab"], case["block"], case["embed"]
    return [V * C, T * C] + case["layers"] * [3 * C * C, C * C, 4 * C * C, 4 * C * C, C, C] + [C]


def work(case):
    if case["kind"] in ("attend", "attend_train"):
        lens = _lengths(case)
        qlens = _query_lengths(case, lens)
        H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
        pairs = sum(q * k - q * (q - 1) // 2 for q, k in zip(qlens, lens))
        rows, keys = 4 * H * D * sum(qlens), 4 * Hk * D * sum(lens)
        if case["kind"] == "attend":
            return {"bytes": 2 * rows + 2 * keys, "flops": 4 * D * H * pairs}
        return {"bytes": 4 * rows + 4 * keys + 4 * H * sum(qlens), "flops": 14 * D * H * pairs}
    if case["kind"] == "adamw":
        n = sum(_sizes(case))
        return {"bytes": n * (28 if case["bits"] == 32 else 16 + 4 / BLOCK), "flops": 20 * n}
    # Rows without a target (the first third) are not read; their gradient is written.
    rows, read = sum(_lengths(case)), sum(n - -(-n // 3) for n in _lengths(case))
    return {"bytes": 4 * case["vocab"] * (read + (rows if case["kind"] == "prefer" else 0)) + 4 * rows, "flops": 5 * read * case["vocab"]}


# ---- inputs ------------------------------------------------------------------------------------

class _Inputs:
    """Seeded inputs made on the GPU, in one fixed order."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)

    def normal(self, *shape, std=1.0):
        return torch.randn(*shape, generator=self.g, device="cuda").mul_(std)

    def uniform(self, *shape):
        return torch.rand(*shape, generator=self.g, device="cuda")


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _starts(lens):
    off = [0]
    for n in lens:
        off.append(off[-1] + n)
    return off


def _prepare_attend(case, r):
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    lens = _lengths(case)
    qlens = _query_lengths(case, lens)
    n, qoff = len(lens), _starts(qlens)
    rows, width = qoff[-1], (H + 2 * Hk) * D
    s = dict(case=case, qlens=_ints(qlens), klens=_ints(lens), q_off=_ints(qoff), most=(max(qlens), max(lens)),
             seq_of=torch.repeat_interleave(torch.arange(n, device="cuda"), _ints(qlens, torch.int64), output_size=rows))
    s["pos_of"] = torch.arange(rows, device="cuda") - s["q_off"].long()[s["seq_of"]]
    s["qkv"] = r.normal(rows, width)  # rows of the QKV product: queries, keys, values
    s["q"] = s["qkv"][:, :H * D].unflatten(1, (H, D))
    if case["cache"]:
        T = case["cache"]
        s["k"], s["v"] = r.normal(n, Hk, T, D), r.normal(n, Hk, T, D)
        s["k_off"], s["k_rows"] = _ints([i * Hk * T for i in range(n + 1)]), n * Hk * T
        s["k_len"], s["k_strides"] = s["klens"], (D, T * D)
    elif case["new"]:
        koff = _starts(lens)
        s["k"], s["v"] = r.normal(koff[-1], Hk, D), r.normal(koff[-1], Hk, D)
        s["k_off"], s["k_rows"], s["k_len"], s["k_strides"] = _ints(koff), koff[-1], None, (Hk * D, D)
    else:
        s["k"], s["v"] = (s["qkv"][:, (H + i * Hk) * D:(H + (i + 1) * Hk) * D].unflatten(1, (Hk, D)) for i in (0, 1))
        s["k_off"], s["k_rows"], s["k_len"], s["k_strides"] = s["q_off"], rows, None, (width, D)
    s["out"] = torch.zeros(rows, H * D, device="cuda")
    if case["kind"] == "attend_train":
        s["dout"] = r.normal(rows, H * D, std=0.1)
        s["lse"], s["dqkv"] = torch.zeros(H, rows, device="cuda"), torch.zeros(rows, width, device="cuda")
    return s


def _prepare_prefer(case, r):
    lens, V = _lengths(case), case["vocab"]
    off = _starts(lens)
    rows = off[-1]
    s = dict(case=case, off=_ints(off), rows=rows, logits=r.normal(rows, V, std=2.0))
    s["seq_of"] = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), _ints(lens, torch.int64), output_size=rows)
    ids = (r.uniform(rows) * V).long().clamp_(max=V - 1)
    # The prompt's rows (about a third) have no target; the others favour it a little.
    answer = (torch.arange(rows, device="cuda") - s["off"].long()[s["seq_of"]]) * 3 >= _ints(lens)[s["seq_of"]]
    s["target"] = torch.where(answer, ids, -1).float()
    s["logits"].scatter_add_(1, ids[:, None], torch.full((rows, 1), 2.0, device="cuda"))
    about = torch.zeros(len(lens), device="cuda").index_add_(0, s["seq_of"], answer.float())
    s["ref"] = -about * math.log(V) + r.normal(len(lens), std=4.0)
    s["grad"], s["logp"], s["loss"] = torch.zeros_like(s["logits"]), torch.zeros(len(lens), device="cuda"), torch.zeros(1, device="cuda")
    return s


def _prepare_adamw(case, r):
    sizes = _sizes(case)
    # Each tensor starts at a multiple of 256 elements of one arena, as an allocator places it; zeros between.
    at = _starts([-(-n // BLOCK) for n in sizes])
    blocks = at[-1]
    s = dict(case=case, sizes=sizes, at=at, tensor_of=torch.repeat_interleave(
        torch.arange(len(sizes), device="cuda"), _ints([b - a for a, b in zip(at, at[1:])], torch.int64), output_size=blocks))
    s["block_in"] = torch.arange(blocks, device="cuda") - _ints(at, torch.int64)[s["tensor_of"]]
    live = (s["block_in"] * BLOCK)[:, None] + torch.arange(BLOCK, device="cuda") < _ints(sizes, torch.int64)[s["tensor_of"]][:, None]
    std = torch.exp(r.normal(blocks, 1, std=1.5)) * 1e-4  # gradients of different blocks differ in size
    s["p"] = r.normal(blocks, BLOCK, std=0.02) * live
    s["g"] = r.normal(blocks, BLOCK) * std * live
    m, root = r.normal(blocks, BLOCK) * (0.3 * std) * live, std * torch.exp(r.normal(blocks, BLOCK, std=0.5)) * live
    if case["bits"] == 32:
        s["m"], s["v"] = m, root * root
    else:
        half = torch.full((blocks, BLOCK), 1 << 15, dtype=torch.int32, device="cuda")
        s["m"], s["me"] = _encode(m, half)
        s["v"], s["ve"] = _encode(root, half, True)
    return s


def prepare(case, seed):
    r = _Inputs(seed)
    if case["kind"] in ("attend", "attend_train"):
        return _prepare_attend(case, r)
    return _prepare_adamw(case, r) if case["kind"] == "adamw" else _prepare_prefer(case, r)


# ---- attention ---------------------------------------------------------------------------------

def _padded(s, x, off, lens, most):
    """Rows [sequence][position][head][dim] of a packed x, positions behind a sequence taking its last row."""
    pos = torch.minimum(torch.arange(most, device="cuda"), (lens.long() - 1).clamp(min=0)[:, None])
    return x[off.long()[:-1, None] + pos]


def _heads(s):
    """q, k, v as [sequence][key head][rows][dim], a key head's query heads one behind the other."""
    c, (mq, mk) = s["case"], s["most"]
    G = c["heads"] // c["kv_heads"]
    q = _padded(s, s["q"], s["q_off"], s["qlens"], mq).unflatten(2, (c["kv_heads"], G))
    q = q.permute(0, 2, 3, 1, 4).flatten(2, 3)
    if c["cache"]:
        return q, s["k"][:, :, :mk], s["v"][:, :, :mk]
    return (q,) + tuple(_padded(s, x, s["k_off"], s["klens"], mk).permute(0, 2, 1, 3).contiguous() for x in (s["k"], s["v"]))


def _visible(s):
    """[sequence][1][1][query][key]: keys up to the query's own position, counted from the ends."""
    mq, mk = s["most"]
    i, j = torch.arange(mq, device="cuda")[:, None], torch.arange(mk, device="cuda")
    ql, kl = s["qlens"].long()[:, None, None], s["klens"].long()[:, None, None]
    return ((j <= i + kl - ql) & (i < ql))[:, None, None]


def _unpadded(s, x):
    """Packed rows of [sequence][key head][head in group x position][dim]."""
    c, G = s["case"], s["case"]["heads"] // s["case"]["kv_heads"]
    x = x.unflatten(2, (G, s["most"][0])).permute(0, 3, 1, 2, 4).flatten(2, 3)
    return x[s["seq_of"], s["pos_of"]].flatten(1)


def _attention_plain(s):
    c = s["case"]
    scale, G = 1.0 / math.sqrt(c["dim"]), c["heads"] // c["kv_heads"]
    q, k, v = _heads(s)
    scores = (torch.matmul(q, k.transpose(2, 3).contiguous()) * scale).unflatten(2, (G, s["most"][0]))
    scores = torch.where(_visible(s), scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    p = (p / torch.where(total == 0, 1.0, total)).flatten(2, 3)
    out = torch.matmul(p, v)
    s["out"].copy_(_unpadded(s, out))
    if c["kind"] == "attend":
        return {"out": s["out"]}
    lse = (top + torch.log(total)).flatten(2, 3)
    s["lse"].copy_(_unpadded(s, lse).t())
    dout = _padded(s, s["dout"].unflatten(1, (c["heads"], c["dim"])), s["q_off"], s["qlens"], s["most"][0])
    dout = dout.unflatten(2, (c["kv_heads"], G)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    dp = torch.matmul(dout, v.transpose(2, 3).contiguous())
    ds = p * (dp - (dout * out).sum(-1, keepdim=True)) * scale
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q)
    dv = torch.matmul(p.transpose(2, 3).contiguous(), dout)
    HD, KD = c["heads"] * c["dim"], c["kv_heads"] * c["dim"]
    s["dqkv"][:, :HD] = _unpadded(s, dq)
    for at, x in ((HD, dk), (HD + KD, dv)):
        s["dqkv"][:, at:at + KD] = x.permute(0, 2, 1, 3)[s["seq_of"], s["pos_of"]].flatten(1)
    return {"out": s["out"], "lse": s["lse"], "dqkv": s["dqkv"]}


def _attention_own(s):
    import freeml_amd as fh

    c = s["case"]
    train = c["kind"] == "attend_train"
    if "shape" not in s:
        H, D = c["heads"], c["dim"]
        rs, hs = s["k_strides"]
        s["shape"] = fh.PackedAttention(
            n_seq=c["seqs"], q_rows=s["qkv"].shape[0], k_rows=s["k_rows"], n_head=H, n_kv_head=c["kv_heads"], head_dim=D,
            scale=1.0 / math.sqrt(D), q_off=s["q_off"].data_ptr(), k_off=s["k_off"].data_ptr(),
            k_len=s["k_len"].data_ptr() if s["k_len"] is not None else None, q_rs=s["qkv"].shape[1], o_rs=H * D,
            k_rs=rs, v_rs=rs, k_hs=hs, v_hs=hs)
        s["ws"] = torch.empty(max(1, fh.attention_packed_workspace(s["shape"], train)), device="cuda")
    a, ws, n = s["shape"], s["ws"].data_ptr(), s["ws"].numel()
    q, k, v, out = (s[x].data_ptr() for x in ("q", "k", "v", "out"))
    if not train:
        fh.attention_packed(a, out, 0, q, k, v, ws, n)
        return {"out": s["out"]}
    lse, dq = s["lse"].data_ptr(), s["dqkv"].data_ptr()
    dk = dq + 4 * c["heads"] * c["dim"]
    dv = dk + 4 * c["kv_heads"] * c["dim"]
    fh.attention_packed(a, out, lse, q, k, v, ws, n)
    fh.attention_packed_backward(a, dq, dk, dv, s["dout"].data_ptr(), out, lse, q, k, v, ws, n)
    return {"out": s["out"], "lse": s["lse"], "dqkv": s["dqkv"]}


def _attention_exact(case, seed):
    s = prepare(case, seed)
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    G, scale = H // Hk, 1.0 / math.sqrt(D)
    qoff, koff = s["q_off"].tolist(), s["k_off"].tolist()
    rows, train = s["qkv"].shape[0], case["kind"] == "attend_train"
    out, lse = torch.zeros(rows, H, D, dtype=torch.float64, device="cuda"), torch.zeros(H, rows, dtype=torch.float64, device="cuda")
    dq, dk, dv = torch.zeros_like(out), torch.zeros(rows, Hk, D, dtype=torch.float64, device="cuda"), torch.zeros(rows, Hk, D, dtype=torch.float64, device="cuda")
    for b, (ql, kl) in enumerate(zip(s["qlens"].tolist(), s["klens"].tolist())):
        a = slice(qoff[b], qoff[b] + ql)
        hidden = torch.arange(kl, device="cuda") > torch.arange(ql, device="cuda")[:, None] + kl - ql
        for h in range(H):
            q = s["q"][a, h].double()
            if case["cache"]:
                k, v = s["k"][b, h // G, :kl].double(), s["v"][b, h // G, :kl].double()
            else:
                k, v = (s[x][koff[b]:koff[b] + kl, h // G].double() for x in ("k", "v"))
            x = (q @ k.T * scale).masked_fill_(hidden, -math.inf)
            lse[h, a] = torch.logsumexp(x, 1)
            p = torch.exp(x - lse[h, a][:, None])
            out[a, h] = p @ v
            if train:
                g = s["dout"][a, h * D:(h + 1) * D].double()
                ds = p * (g @ v.T - (g * out[a, h]).sum(1, keepdim=True)) * scale
                dq[a, h] = ds @ k
                dk[a, h // G] += ds.T @ q
                dv[a, h // G] += p.T @ g
    if not train:
        return {"out": out.flatten(1)}
    return {"out": out.flatten(1), "lse": lse, "dqkv": torch.cat([x.flatten(1) for x in (dq, dk, dv)], 1)}


# ---- preference loss ---------------------------------------------------------------------------

BETA = 0.1


def _prefer_plain(s):
    c, z = s["case"], s["logits"]
    ids = s["target"].long()
    valid = ids >= 0
    ids = ids.clamp(min=0)[:, None]
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    row = (z.gather(1, ids) - top).double() - torch.log(total.double())
    upto = torch.cat([torch.zeros(1, dtype=torch.float64, device="cuda"), torch.cumsum(row[:, 0] * valid, 0)])[s["off"].long()]
    logp = upto[1:] - upto[:-1]
    s["logp"].copy_(logp)
    if c["kind"] == "logprobs":
        return {"logp": s["logp"]}
    ratio = logp - s["ref"].double()
    x, eps = BETA * (ratio[0::2] - ratio[1::2]), c["smoothing"]
    soft = lambda y: torch.clamp(y, min=0) + torch.log1p(torch.exp(-torch.abs(y)))  # noqa: E731
    s["loss"].copy_(((1 - eps) * soft(-x) + eps * soft(x)).mean())
    f = BETA / c["pairs"] * ((1 - eps) / (1 + torch.exp(x)) - eps / (1 + torch.exp(-x)))
    f = torch.stack([f, -f], 1).flatten()[s["seq_of"]] * valid
    torch.mul(e, (-f[:, None] / total.double()).float(), out=s["grad"])
    s["grad"].scatter_add_(1, ids, f[:, None].float())
    return {"grad": s["grad"], "loss": s["loss"], "logp": s["logp"]}


def _prefer_own(s):
    import freeml_amd as fh

    c, rows, V = s["case"], s["rows"], s["case"]["vocab"]
    if "ws" not in s:
        s["ws"] = torch.empty(fh.preference_workspace(rows, 2 * c["pairs"]), device="cuda")
    p = {x: s[x].data_ptr() for x in ("ws", "target", "logits", "off", "logp", "grad", "loss", "ref")}
    if c["kind"] == "logprobs":
        fh.sequence_logprobs(p["logp"], p["ws"], p["target"], p["logits"], p["off"], V, rows, 2 * c["pairs"])
        return {"logp": s["logp"]}
    fh.preference_logits(p["grad"], p["loss"], p["logp"], p["ws"], p["target"], p["logits"], p["off"], p["ref"], V, rows,
                         c["pairs"], BETA, c["smoothing"])
    return {"grad": s["grad"], "loss": s["loss"], "logp": s["logp"]}


def _prefer_exact(case, seed):
    s = prepare(case, seed)
    off, ids = s["off"].tolist(), s["target"].long()
    logp, parts = [], []
    for a, b in zip(off, off[1:]):
        t = ids[a:b]
        row = torch.log_softmax(s["logits"][a:b].double(), 1)
        logp.append(row.gather(1, t.clamp(min=0)[:, None])[:, 0][t >= 0].sum())
    logp = torch.stack(logp)
    if case["kind"] == "logprobs":
        return {"logp": logp}
    x = (BETA * ((logp[0::2] - s["ref"][0::2].double()) - (logp[1::2] - s["ref"][1::2].double()))).requires_grad_(True)
    eps = case["smoothing"]
    loss = -((1 - eps) * torch.nn.functional.logsigmoid(x) + eps * torch.nn.functional.logsigmoid(-x)).mean()
    loss.backward()
    for i, (a, b) in enumerate(zip(off, off[1:])):
        t = ids[a:b]
        part = torch.softmax(s["logits"][a:b].double(), 1).neg_()
        part.scatter_add_(1, t.clamp(min=0)[:, None], torch.ones(b - a, 1, dtype=torch.float64, device="cuda"))
        parts.append(part * (t >= 0)[:, None] * (-BETA * x.grad[i // 2] * (1 if i % 2 == 0 else -1)))
    return {"grad": torch.cat(parts), "loss": loss.detach().reshape(1), "logp": logp}


# ---- AdamW -------------------------------------------------------------------------------------

LR, B1, B2, EPS, DECAY, SEED = 3e-4, 0.9, 0.999, 1e-8, 0.1, 12345
F32 = lambda x: torch.tensor(x, dtype=torch.float32).item()  # noqa: E731


def _powers(case):
    return F32(F32(B1) ** case["step"]), F32(F32(B2) ** case["step"])


def _encode(x, rnd, square=False):
    """Blocks of values -> e4m3 codes (exponent 1 .. 15 of bias 7, three mantissa bits; sign on top) of
    x / 2^(E - 127) and the blocks' E: the largest value lands in [2^7, 2^8).  A value between two codes goes
    up where its 16 bits of rnd, as a fraction, are below its share of the gap; square: the square's share
    of the gap between the codes' squares."""
    E = ((x.abs().view(torch.int32).amax(1) >> 23) - 7).clamp(min=1)
    y = x.abs() * ((254 - E) << 23).view(torch.float32)[:, None]
    bits, normal = y.view(torch.int32), y >= 2.0**-6
    small = torch.floor(y * 512.0)
    low = torch.where(normal, (bits & -(1 << 20)).view(torch.float32), small * 2.0**-9)
    high = torch.where(normal, ((bits & -(1 << 20)) + (1 << 20)).view(torch.float32), low + 2.0**-9)
    gap, rest = high - low, y - low
    if square:
        gap, rest = gap * (high + low), rest * (y + low)
    code = torch.where(normal, (bits >> 20) - (120 << 3), small.to(torch.int32)) + (rnd.float() * 2.0**-16 * gap < rest)
    return (code | torch.where(x < 0, 128, 0)).to(torch.uint8), E.to(torch.uint8)


def _decode(code, E):
    return code.view(torch.float8_e4m3fn).float() * (E.to(torch.int32) << 23).view(torch.float32)[:, None]


def _mix32(h):
    h = (h ^ (h >> 16)) * 0x85EBCA6B & 0xFFFFFFFF
    h = (h ^ (h >> 13)) * 0xC2B2AE35 & 0xFFFFFFFF
    return h ^ (h >> 16)


def _random(s):
    """32 random bits per element, from the seed, the tensor's number and the element's."""
    key = _mix32(torch.full((), (SEED & 0xFFFFFFFF) ^ 0x9E3779B9, dtype=torch.int64, device="cuda"))
    key = _mix32(key ^ (s["tensor_of"] + (SEED >> 32) & 0xFFFFFFFF))
    i = (s["block_in"] * BLOCK)[:, None] + torch.arange(BLOCK, device="cuda")
    return _mix32((i & 0xFFFFFFFF) ^ (key ^ (i[:, :1] >> 32).squeeze(1) * 0x9E3779B9 & 0xFFFFFFFF)[:, None])


def _adamw_plain(s):
    c, g, p = s["case"], s["g"], s["p"]
    b1, b2, lr = F32(B1), F32(B2), F32(LR)
    # Divisors as device values: torch turns a division by a number into a product with its inverse.
    d1, d2 = (torch.full((), F32(1 - x), device="cuda") for x in _powers(c))
    if c["bits"] == 32:
        m, v = s["m"], s["v"]
    else:
        m, root = _decode(s["m"], s["me"]), _decode(s["v"], s["ve"])
        v = root * root
    m = m * b1 + g * F32(1 - b1)
    v = v * b2 + g * F32(1 - b2) * g
    update = (m / d1) * lr / (torch.sqrt(v / d2) + F32(EPS))
    p.copy_((p + update) - p * F32(lr * F32(DECAY)))
    if c["bits"] == 32:
        s["m"].copy_(m)
        s["v"].copy_(v)
        return {"p": p, "m": s["m"], "v": s["v"]}
    rnd, root = _random(s), torch.sqrt(v)
    code, E = _encode(m, (rnd & 0xFFFF).to(torch.int32))
    s["m"].copy_(code)
    s["me"].copy_(E)
    code, E = _encode(root, (rnd >> 16).to(torch.int32), True)
    s["v"].copy_(torch.where(root > 0, code.clamp(min=1), code))
    s["ve"].copy_(E)
    return _adamw_states(s)


def _adamw_states(s):
    """8-bit states as the values their codes stand for, in units of their block's scale, and the scales' exponents."""
    return {"p": s["p"], "m": s["m"].view(torch.float8_e4m3fn), "v": s["v"].view(torch.float8_e4m3fn), "me": s["me"], "ve": s["ve"]}


def _adamw_own(s):
    import freeml_amd as fh

    c = s["case"]
    if "table" not in s:
        size = 4 if c["bits"] == 32 else 1
        place = lambda x, a, n: s[x].data_ptr() + a * BLOCK * n  # noqa: E731
        s["table"] = fh.adamw_tensors([
            (place("p", a, 4), place("g", a, 4), place("m", a, size), place("v", a, size), n) +
            (() if size == 4 else (s["me"].data_ptr() + a, s["ve"].data_ptr() + a)) for a, n in zip(s["at"], s["sizes"])])
    fh.adamw_update_multi(s["table"], c["bits"], LR, B1, B2, *_powers(c), EPS, DECAY, SEED)
    return {"p": s["p"], "m": s["m"], "v": s["v"]} if c["bits"] == 32 else _adamw_states(s)


def _adamw_exact(case, seed):
    s = prepare(case, seed)
    d = torch.float64
    p1, p2 = _powers(case)
    b1, b2 = F32(B1), F32(B2)

    def value(x, e):
        x = x.to(torch.int64)
        ex, ma = x >> 3 & 15, x & 7
        v = torch.where(ex > 0, (8 + ma).to(d) * torch.pow(2.0, (ex - 10).to(d)), ma.to(d) * 2.0**-9)
        return torch.where(x > 127, -v, v) * torch.pow(2.0, e.to(d) - 127)[:, None]

    def stored(x, rnd, power):
        ex = torch.floor(torch.log2(x.abs().amax(1, keepdim=True))) - 7  # the block's unit, a power of two
        ex = torch.where(torch.isfinite(ex), ex, -126.0).clamp(min=-126)
        y = x.abs() * torch.pow(2.0, -ex)
        step = torch.pow(2.0, torch.floor(torch.log2(y.clamp(min=2.0**-6))) - 3)
        low = torch.floor(y / step) * step
        share = (y**power - low**power) / ((low + step) ** power - low**power)
        return torch.sign(x) * torch.where((rnd.to(d) / 65536 < share), low + step, low)

    g = s["g"].double()
    m, v = (s["m"].double(), s["v"].double()) if case["bits"] == 32 else (value(s["m"], s["me"]), value(s["v"], s["ve"]) ** 2)
    m = b1 * m + F32(1 - b1) * g
    v = b2 * v + F32(1 - b2) * g * g
    p = s["p"].double()
    p = p + F32(LR) * (m / (1 - p1)) / (torch.sqrt(v / (1 - p2)) + F32(EPS)) - F32(LR) * F32(DECAY) * p
    if case["bits"] == 32:
        return {"p": p, "m": m, "v": v}
    rnd = _random(s)
    root = stored(torch.sqrt(v), rnd >> 16, 2)
    return {"p": p, "m": stored(m, rnd & 0xFFFF, 1), "v": torch.where(v > 0, root.clamp(min=2.0**-9), root), "me": None, "ve": None}


# ------------------------------------------------------------------------------------------------

def run(state):
    kind = state["case"]["kind"]
    if kind in ("attend", "attend_train"):
        return _attention_own(state) if own else _attention_plain(state)
    if kind == "adamw":
        return _adamw_own(state) if own else _adamw_plain(state)
    return _prefer_own(state) if own else _prefer_plain(state)


def exact(case, seed):
    if case["kind"] in ("attend", "attend_train"):
        return _attention_exact(case, seed)
    return _adamw_exact(case, seed) if case["kind"] == "adamw" else _prefer_exact(case, seed)
