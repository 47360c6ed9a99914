"""The paged key/value operators as a user calls them, and their plain forms in torch.

Three operators of one cache: `append` rotates new queries and keys and writes keys and
values into the cache's pages, `decode` attends from one new token per sequence, and
`prefill` attends from a ragged batch of prompt pieces whose keys are in the cache
already.  Pages are [pages][kv heads][page][dim] in any order of the first three; a
sequence's position t lives in page table[seq][t // page] at row t % page.

A key at position j is visible to the query at position p when j is below the sequence's
length and either j <= p, with p - j < window where a window is set, or j < prefix.  The
score is scale * q.k, then cap * tanh(score / cap) where a cap is set, then
- slope[head] * |p - j| where slopes are set.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def _case(name, op, **more):
    c = {"name": name, "op": op, "type": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "seqs": 1,
         "len_lo": 1, "len_hi": 1, "q_lo": 1, "q_hi": 1, "by_token": False, "interleaved": False, "in_type": "bf16",
         "window": 0, "prefix": 0, "cap": 0.0, "slopes": False}
    c.update(more)
    return c


def listed():
    return [
        # the new token of the one sequence that a command-line user talks to: fp32
        # activations of the 14-head model into its cache; latency is all
        _case("append-one", "append", heads=14, kv_heads=2, dim=64, in_type="f32", len_lo=777, len_hi=777),
        # the prompts of three users arrive at once; interleaved pairs, pages of 64
        _case("append-16k", "append", page=64, seqs=3, len_lo=16, len_hi=9001, q_lo=15, q_hi=9001,
              interleaved=True),
        # one sequence of the fp32 engine, 777 positions: latency
        _case("decode-one-f32", "decode", type="f32", heads=14, kv_heads=2, dim=64, len_lo=777, len_hi=777),
        # a serving batch of the 32-head, 64-wide model, sequences of every age
        _case("decode-64", "decode", dim=64, page=32, seqs=64, len_lo=1, len_hi=2047),
        # two readers of long documents: few heads, so the length is what can be split
        _case("decode-long", "decode", type="f16", heads=12, kv_heads=2, page=64, seqs=2, len_lo=40001,
              len_hi=131071),
        # a full card: 128 sequences, pages ordered [page][token][head]
        _case("decode-128", "decode", seqs=128, len_lo=500, len_hi=8192, by_token=True),
        # the same kind of batch under a sliding window with four kept first tokens and
        # capped scores
        _case("decode-window", "decode", type="f16", page=32, seqs=40, len_lo=3, len_hi=16001, window=1024, prefix=4,
              cap=30.0),
        # five short pieces after cached text in the fp32 engine
        _case("prefill-f32", "prefill", type="f32", heads=14, kv_heads=2, dim=64, seqs=5, len_lo=1, len_hi=601,
              q_lo=1, q_hi=70),
        # the 1024-token prompt of the 14-head model
        _case("prefill-1024", "prefill", heads=14, kv_heads=2, dim=64, len_lo=1024, len_hi=1024, q_lo=1024,
              q_hi=1024),
        # a short question about a long cached text
        _case("prefill-extend", "prefill", heads=12, kv_heads=2, page=64, seqs=2, len_lo=65537, len_hi=65537, q_lo=16,
              q_hi=17),
        # a long prompt from nothing
        _case("prefill-8k", "prefill", page=64, len_lo=8192, len_hi=8192, q_lo=8192, q_hi=8192),
        # ragged pieces with every option of the scores
        _case("prefill-options", "prefill", type="f16", page=32, seqs=6, len_lo=40, len_hi=4097, q_lo=33, q_hi=1500,
              window=700, prefix=129, cap=50.0, slopes=True, by_token=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        for k in w:
            most[k] = max(most.get(k, 0), w[k])
    while True:
        op = rng.choice(["append", "decode", "decode", "prefill", "prefill"])
        heads, kv_heads = rng.choice([(14, 2), (32, 8), (12, 2), (8, 8), (16, 1), (5, 5), (40, 4)])
        c = _case("", op, type=rng.choice(["f32", "f16", "bf16", "bf16"]), heads=heads, kv_heads=kv_heads,
                  dim=rng.choice([32, 64, 96, 128, 128]), page=rng.choice([8, 16, 24, 32, 64, 128]),
                  by_token=rng.random() < 0.5, interleaved=rng.random() < 0.5)
        del c["name"]
        c["in_type"] = rng.choice([c["type"], "f32"])
        if rng.random() < 0.3:
            c["window"] = _log_int(rng, 1, 4000)
        if rng.random() < 0.3:
            c["prefix"] = _log_int(rng, 1, 500)
        if rng.random() < 0.3:
            c["cap"] = rng.choice([20.0, 30.0, 50.0])
        c["slopes"] = rng.random() < 0.3
        if op == "decode":
            c["seqs"] = _log_int(rng, 1, 200)
            c["len_hi"] = _log_int(rng, 1, 131071)
            c["len_lo"] = _log_int(rng, 1, c["len_hi"])
        else:
            c["seqs"] = _log_int(rng, 1, 12)
            c["q_hi"] = _log_int(rng, 1, 8192 if op == "prefill" else 12000)
            c["q_lo"] = _log_int(rng, 1, c["q_hi"])
            c["len_lo"] = c["q_hi"] + _log_int(rng, 1, 4000) - 1
            c["len_hi"] = c["len_lo"] + _log_int(rng, 1, 30000) - 1
        w = work(c)
        queries = c["q_hi"] if op == "prefill" else 1
        padded = c["seqs"] * c["len_hi"] * max(c["kv_heads"] * c["dim"], c["heads"] * queries)
        limit = 64 * 2 ** 20 if c["type"] == "f32" and op == "prefill" else 2 ** 31
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"] and (op == "append" or padded <= limit):
            return c


def _lengths(c):
    """The sequences' (new rows, length) of a case: its extremes and a spread between them."""
    rs = np.random.RandomState(c["seqs"] * 7 + c["len_hi"] % 1000)
    n = c["seqs"]
    f = np.sort(rs.rand(n))
    f[0], f[-1] = 0.0, 1.0
    q = np.round(c["q_lo"] + (c["q_hi"] - c["q_lo"]) * f).astype(np.int64)
    length = np.round(c["len_lo"] + (c["len_hi"] - c["len_lo"]) * f).astype(np.int64)
    if c["op"] == "decode":
        q[:] = 1
    return q, np.maximum(length, q)


def _visible(c):
    """Keys that a case's queries see, per sequence: (summed over the queries, of any query)."""
    pairs, keys = [], []
    for q, length in zip(*_lengths(c)):
        p = np.arange(length - q, length)
        low = np.maximum(p - c["window"] + 1, 0) if c["window"] else np.zeros_like(p)
        pre = min(c["prefix"], int(length))
        pairs.append(int(np.sum(p + 1 - low + np.minimum(low, pre) + np.maximum(pre - (p + 1), 0))))
        keys.append(int(min(length, length - low[0] + min(low[0], pre))))
    return pairs, keys


def work(case):
    c = case
    q, _ = _lengths(c)
    rows, item, d = int(q.sum()), BYTES[c["type"]], c["dim"]
    if c["op"] == "append":  # q, k, v read; q and the pages' rows written; a table row of angles for each token
        b = rows * d * ((c["heads"] + 2 * c["kv_heads"]) * (BYTES[c["in_type"]] + item) + 4)
        return {"bytes": b, "flops": rows * d * 3 * (c["heads"] + c["kv_heads"])}
    pairs, keys = _visible(c)
    return {"bytes": 2 * rows * c["heads"] * d * item + 2 * sum(keys) * c["kv_heads"] * d * item,
            "flops": 4 * sum(pairs) * c["heads"] * d}


def prepare(case, seed):
    c, dev = case, "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    rs = np.random.RandomState(seed % (2 ** 31))
    q, length = _lengths(c)
    order = rs.permutation(c["seqs"])
    q, length = q[order], length[order]
    rows, page, kv, d, dt = int(q.sum()), c["page"], c["kv_heads"], c["dim"], TYPES[c["type"]]

    def normal(*shape, dtype=dt, scale=1.0):
        return torch.empty(shape, device=dev, dtype=dtype).normal_(0, scale, generator=g)

    need = -(-length // page)
    pages = int(need.sum()) + 3
    if c["by_token"]:
        k, v = (normal(pages, page, kv, d).transpose(1, 2) for _ in range(2))
    else:
        k, v = (normal(pages, kv, page, d) for _ in range(2))
    ids = rs.permutation(pages)
    table = np.zeros((c["seqs"], int(need.max())), np.int32)
    at = 0
    for i, m in enumerate(need):
        table[i, :m] = ids[at:at + m]
        at += m
    s = {"case": dict(c), "k": k, "v": v, "table": torch.from_numpy(table).to(dev),
         "kv_len": torch.from_numpy(length.astype(np.int32)).to(dev),
         "q_start": torch.from_numpy(np.concatenate([[0], np.cumsum(q)]).astype(np.int32)).to(dev),
         "q_max": int(q.max()), "rows": rows}
    if c["op"] == "append":
        seq = np.repeat(np.arange(c["seqs"]), q)
        pos = np.concatenate([np.arange(b - a, b) for a, b in zip(q, length)])
        s["seq"] = torch.from_numpy(seq.astype(np.int32)).to(dev)
        s["pos"] = torch.from_numpy(pos.astype(np.int32)).to(dev)
        qkv = normal(rows, c["heads"] + 2 * kv, d, dtype=TYPES[c["in_type"]])
        s["new"] = qkv.split([c["heads"], kv, kv], dim=1)
        i = torch.arange(d // 2, device=dev, dtype=torch.float64)
        angle = torch.arange(int(length.max()), device=dev, dtype=torch.float64)[:, None] * 10000.0 ** (-2 * i / d)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["q_out"] = torch.empty(rows, c["heads"], d, device=dev, dtype=dt)
    else:
        s["q"] = normal(rows, c["heads"], d, scale=1.5)
        s["out"] = torch.empty_like(s["q"])
        s["prefix"] = None
        if c["prefix"]:
            s["prefix"] = torch.full((c["seqs"],), c["prefix"], device=dev, dtype=torch.int32)
        s["slopes"] = None
        if c["slopes"]:
            s["slopes"] = 2.0 ** (-8.0 * (torch.arange(c["heads"], device=dev) + 1) / c["heads"]).float()
    return s


def _append(s):
    c = s["case"]
    q, k, v = (t.float() for t in s["new"])
    at = s["pos"].long()
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]

    def rotate(x):
        if c["interleaved"]:
            a, b = x[..., 0::2], x[..., 1::2]
            return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
        a, b = x.chunk(2, -1)
        return torch.cat((a * cos - b * sin, a * sin + b * cos), -1)

    where = s["table"][s["seq"].long(), at // c["page"]].long()
    s["k"][where, :, at % c["page"]] = rotate(k).to(s["k"].dtype)
    s["v"][where, :, at % c["page"]] = v.to(s["v"].dtype)
    return {"q": rotate(q).to(s["k"].dtype), "k": s["k"], "v": s["v"]}


def _attend(s):
    c = s["case"]
    seqs, kv, d, heads = c["seqs"], c["kv_heads"], c["dim"], c["heads"]
    group, most = heads // kv, s["q_max"]
    k, v = (s[n][s["table"].long()].transpose(1, 2).reshape(seqs, kv, -1, d).float() for n in "kv")
    start, length = s["q_start"].long(), s["kv_len"].long()
    count = start[1:] - start[:-1]
    i = torch.arange(most, device=k.device)
    there = i[None] < count[:, None]
    q = torch.zeros(seqs, most, heads, d, device=k.device)
    q[there] = s["q"].float()
    q = q.view(seqs, most, kv, group, d).permute(0, 2, 3, 1, 4).reshape(seqs, kv, group * most, d)
    x = (q @ k.transpose(-1, -2)).view(seqs, kv, group, most, -1) * d ** -0.5
    if c["cap"]:
        x = c["cap"] * torch.tanh(x / c["cap"])
    j = torch.arange(x.shape[-1], device=k.device)
    p = (length - count)[:, None] + i[None]
    away = p[:, :, None] - j
    if s["slopes"] is not None:
        x = x - s["slopes"].view(1, kv, group, 1, 1) * away[:, None, None].abs()
    seen = away >= 0
    if c["window"]:
        seen &= away < c["window"]
    if s["prefix"] is not None:
        seen |= j < s["prefix"].long()[:, None, None]
    seen &= j < length[:, None, None]
    x = torch.where(seen[:, None, None], x, -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True).clamp_min(-1e30))
    x = x / x.sum(-1, keepdim=True).clamp_min(1e-30)
    o = (x.view(seqs, kv, group * most, -1) @ v).view(seqs, kv, group, most, d)
    return o.permute(0, 3, 1, 2, 4).reshape(seqs, most, heads, d)[there].to(s["q"].dtype)


def run(state):
    s = state
    c = s["case"]
    if not own:
        return _append(s) if c["op"] == "append" else _attend(s)
    cache = s.get("cache")
    if cache is None:
        folder = os.path.join(os.getcwd(), "mocha-moze-llm_b200")
        if folder not in sys.path:
            sys.path.insert(0, folder)
        import mocha_kv
        cache = s["cache"] = mocha_kv.KvPages(s["k"], s["v"])
    if c["op"] == "append":
        q, k, v = s["new"]
        cache.append(q, k, v, s["seq"], s["pos"], s["table"], cos=s["cos"], sin=s["sin"],
                     interleaved=c["interleaved"], q_out=s["q_out"])
        return {"q": s["q_out"], "k": s["k"], "v": s["v"]}
    more = {"window": c["window"], "prefix": s["prefix"], "cap": c["cap"], "slopes": s["slopes"], "out": s["out"]}
    if c["op"] == "decode":
        return cache.decode(s["q"], s["table"], s["kv_len"], **more)
    return cache.prefill(s["q"], s["q_start"], s["table"], s["kv_len"], **more)


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    table, page = s["table"].cpu().numpy(), c["page"]
    if c["op"] == "append":
        seq, pos = s["seq"].cpu().numpy(), s["pos"].cpu().numpy()
        where = torch.from_numpy(table[seq, pos // page].astype(np.int64) * page + pos % page).cuda()
        at = torch.from_numpy(pos.astype(np.int64)).cuda()
        turn = torch.complex(s["cos"].double(), s["sin"].double())[at].unsqueeze(1)

        def rotate(x):
            x = x.double()
            if c["interleaved"]:
                z = torch.view_as_complex(x.reshape(*x.shape[:-1], -1, 2).contiguous()) * turn
                return torch.view_as_real(z).reshape(x.shape)
            half = x.shape[-1] // 2
            z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * turn
            return torch.cat((z.real, z.imag), -1)

        out = {"q": rotate(s["new"][0])}
        for name, rows in (("k", rotate(s["new"][1])), ("v", s["new"][2].double())):
            pool = s[name].double().transpose(1, 2).reshape(-1, c["kv_heads"], c["dim"])
            pool[where] = rows
            out[name] = pool.view(-1, page, c["kv_heads"], c["dim"]).transpose(1, 2)
        return out
    group = c["heads"] // c["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    starts, lengths = s["q_start"].tolist(), s["kv_len"].tolist()
    for b in range(c["seqs"]):
        a, e, n = starts[b], starts[b + 1], lengths[b]
        ids = torch.from_numpy(table[b, :-(-n // page)].astype(np.int64)).cuda()
        for h in range(c["kv_heads"]):
            k, v = (s[x][ids, h].reshape(-1, c["dim"])[:n].double() for x in "kv")
            for lo in range(a, e, 2048):
                hi = min(lo + 2048, e)
                p = torch.arange(n - (e - a) + lo - a, n - (e - a) + hi - a, device="cuda")[:, None]
                j = torch.arange(n, device="cuda")[None]
                hide = j > p
                if c["window"]:
                    hide |= j <= p - c["window"]
                if c["prefix"]:
                    hide &= j >= c["prefix"]
                for m in range(h * group, (h + 1) * group):
                    z = s["q"][lo:hi, m].double() @ k.T / math.sqrt(c["dim"])
                    if c["cap"]:
                        z = torch.tanh(z / c["cap"]) * c["cap"]
                    if c["slopes"]:
                        z -= float(s["slopes"][m]) * (p - j).abs().double()
                    z.masked_fill_(hide, -math.inf)
                    out[lo:hi, m] = torch.softmax(z, -1) @ v
    return out
