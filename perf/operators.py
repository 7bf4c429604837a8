"""The 4-bit operators whose speed this framework answers for: attention over a key/value cache held in 4 bits, the
cache's writing and reading back, and the Linear over 4-bit weights with group scales.

A case is a dict of plain values; `kind` names the operator:

  attention  attention_kv4: new queries against a paged 4-bit cache (`batch` sequences of up to `len` cached
             tokens, the `seq` newest of them with a query)
  cache      kv4_write, then kv4_read of what was written
  read       kv4_read of a cached prefix
  linear     linear_w4

Values in 4 bits are c * s + m with a code c of 0 .. 15 and an fp16 pair (s, m) per group: 32 features of a token
and head in the cache, `group` input features of an output row in a weight.  m is the group's minimum and
s = fp16(fp32(fp32(max - min) / 15)).
"""
import importlib
import math

import torch

own = False
F16, F32, F64 = torch.float16, torch.float32, torch.float64
MASKED = float("-inf")
# nibble of feature f of a 32-bit word (feature pairs lie 16 bits apart)
NIBBLE = [0, 4, 1, 5, 2, 6, 3, 7]


def _att(name, batch, seq, heads, kv, dh, dv, length, page, ragged=False, mask="causal"):
    return {"name": name, "kind": "attention", "batch": batch, "seq": seq, "heads": heads, "kv": kv, "dh_qk": dh,
            "dh_v": dv, "len": length, "page": page, "ragged": ragged, "mask": mask}


def _lin(name, T, inn, out, group, act="none", bias=True):
    return {"name": name, "kind": "linear", "T": T, "in": inn, "out": out, "group": group, "act": act, "bias": bias}


def listed():
    return [
        # one sentence answered token by token: the smallest call, where latency counts
        _att("att-b1-l128", 1, 1, 12, 12, 64, 64, 128, 16),
        # a serving batch of conversations of different lengths
        _att("att-b16-l2000", 16, 1, 16, 16, 64, 64, 2000, 64, ragged=True),
        # a few very long documents, key/value heads shared by four query heads: the memory-bound end
        _att("att-b4-l32768-gqa", 4, 1, 32, 8, 128, 128, 32768, 64),
        # the next 64 tokens of two prompts on top of what is cached
        _att("att-b2-s64-l1025", 2, 64, 12, 12, 64, 64, 1025, 32),
        # a few proposed tokens at once, pruned Q/K features, shared heads, ragged lengths
        _att("att-b7-s3-l777-qk48", 7, 3, 12, 4, 48, 64, 777, 16, ragged=True),
        # a batch of prompts cached and read back
        {"name": "cache-b8-s2048", "kind": "cache", "batch": 8, "seq": 2048, "kv": 16, "dh_qk": 64, "dh_v": 64,
         "page": 64, "start": 0},
        # one new token of each of many conversations
        {"name": "cache-b64-s1", "kind": "cache", "batch": 64, "seq": 1, "kv": 12, "dh_qk": 64, "dh_v": 64,
         "page": 16, "start": 333},
        # a long cached prefix read back for a dense pass over it
        {"name": "read-b4-l8191", "kind": "read", "batch": 4, "seq": 8191, "kv": 8, "dh_qk": 128, "dh_v": 128,
         "page": 64, "start": 1},
        # the fused projection of one token: the smallest product
        _lin("w4-t1-768-2304", 1, 768, 2304, 32),
        # one token through a large matrix: weight bandwidth
        _lin("w4-t1-8192-8192", 1, 8192, 8192, 128, bias=False),
        # a ragged little batch through a feed-forward block's second product
        _lin("w4-t7-4096-1024", 7, 4096, 1024, 64),
        # a prompt through its first product
        _lin("w4-t2000-1024-4096", 2000, 1024, 4096, 128, act="relu"),
    ]


def _log(rng, low, high):
    return min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "linear", "linear", "cache", "read"])
    if kind == "attention":
        kv, ratio = rng.choice([1, 2, 4, 8, 12, 16]), rng.choice([1, 1, 2, 3, 4, 8])
        dh = 16 * rng.randint(1, 8)
        dv = dh if rng.random() < 0.7 else 16 * rng.randint(1, 8)
        seq = 1 if rng.random() < 0.5 else _log(rng, 1, 128)
        batch = _log(rng, 1, 64)
        # no more keys than the long documents have, and no more scores than they or the prompt chunk take
        top = min(32768, 4 * 32768 * 8 * 128 // (batch * kv * max(dh, dv)), 4 * 32 * 32768 // (batch * seq * kv * ratio))
        length = max(seq, _log(rng, 1, max(1, top)))
        c = _att("", batch, seq, kv * ratio, kv, dh, dv, length, rng.choice([16, 32, 64, 128]),
                 rng.random() < 0.5, "causal" if rng.random() < 0.7 else "none")
    elif kind == "linear":
        inn, out = 16 * _log(rng, 1, 512), 16 * _log(rng, 1, 512)
        T = _log(rng, 1, 2048)
        T = max(1, min(T, 2000 * 1024 * 4096 // (inn * out)))
        c = _lin("", T, inn, out, rng.choice([32, 64, 128]), rng.choice(["none", "relu"]), rng.random() < 0.7)
    else:
        kv, dh = rng.choice([1, 2, 4, 8, 12, 16]), 16 * rng.randint(1, 8)
        dv = dh if rng.random() < 0.7 else 16 * rng.randint(1, 8)
        batch = _log(rng, 1, 64)
        most = (8 * 2048 * 16 * 64 if kind == "cache" else 4 * 8191 * 8 * 128) // (batch * kv * max(dh, dv))
        c = {"kind": kind, "batch": batch, "seq": _log(rng, 1, max(1, min(8191, most))), "kv": kv, "dh_qk": dh,
             "dh_v": dv, "page": rng.choice([16, 32, 64, 128]), "start": _log(rng, 1, 500) - 1}
    c.pop("name", None)
    return c


def _groups(case):
    return (max(case["dh_qk"], case["dh_v"]) + 31) // 32


def _lengths(case):
    """Cached tokens of every sequence: `len`, or spread down to half of it."""
    n, seq = case["len"], case["seq"]
    if not case["ragged"]:
        return [n] * case["batch"]
    return [max(seq, n - (b * 37 + b * b * 11) % (n // 2 + 1)) for b in range(case["batch"])]


def _normal(g, shape, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=F32) * std).to(F16)


def _params(g, shape, size):
    """(s, m) of groups whose values are about N(offset, size^2): the codes spread over all sixteen levels."""
    s = size * (0.2 + 0.15 * torch.rand(shape, generator=g, device="cuda", dtype=F32))
    m = -7.5 * s + 0.3 * size * torch.randn(shape, generator=g, device="cuda", dtype=F32)
    return torch.stack([s, m], dim=-1).to(F16)


def _codes(g, shape):
    return torch.randint(0, 256, shape, generator=g, device="cuda", dtype=torch.uint8)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    st = {"case": case}
    if case["kind"] == "linear":
        T, inn, out, group = case["T"], case["in"], case["out"], case["group"]
        nb = (inn + 127) // 128
        st["x"] = _normal(g, (T, inn))
        st["bias"] = _normal(g, (out,), 0.1) if case["bias"] else None
        st["codes"] = _codes(g, (out // 16, nb, 2, 32, 16))
        st["params"] = _params(g, (out // 16, nb, 16, 128 // group), 0.02)
        if own:
            et = importlib.import_module("scpaper-2021_b200")
            st["et"] = et
            st["weight"] = et.W4Weight.from_arrays(st["codes"], st["params"], inn, out, group)
            st["act"] = {"none": et.ACT_NONE, "relu": et.ACT_RELU}[case["act"]]
        return st
    batch, seq, kv, page, ng = case["batch"], case["seq"], case["kv"], case["page"], _groups(case)
    most = case["len"] if case["kind"] == "attention" else case["start"] + seq
    per = (most + page - 1) // page
    pages = batch * per + 3
    st["table"] = torch.randperm(pages, generator=g, device="cuda")[: batch * per].view(batch, per).to(torch.int32)
    if case["kind"] == "cache":  # what the pages held before
        arrays = [torch.zeros((pages, kv, page, 16 * ng), dtype=torch.uint8, device="cuda"),
                  torch.zeros((pages, kv, page, ng, 2), dtype=F16, device="cuda")]
        arrays += [a.clone() for a in arrays]
        # keys have features with an offset of their own, as a projection's bias leaves them
        dh, dv = case["dh_qk"], case["dh_v"]
        st["k"] = (_normal(g, (batch * seq, kv * dh)) + _normal(g, (kv * dh,), 1.5)).contiguous()
        st["v"] = _normal(g, (batch * seq, kv * dv))
    else:
        arrays = [_codes(g, (pages, kv, page, 16 * ng)), _params(g, (pages, kv, page, ng), 1.0),
                  _codes(g, (pages, kv, page, 16 * ng)), _params(g, (pages, kv, page, ng), 1.0)]
    if case["kind"] == "attention":
        st["q"] = _normal(g, (batch * seq, case["heads"] * case["dh_qk"]))
        st["kv_len"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
    else:
        st["start"] = torch.full((batch,), case["start"], dtype=torch.int32, device="cuda")
    if own:
        et = importlib.import_module("scpaper-2021_b200")
        cache = et.KV4Cache(pages, page, kv, case["dh_qk"], case["dh_v"], device="cuda")
        for mine, made in zip((cache.k_codes, cache.k_params, cache.v_codes, cache.v_params), arrays):
            mine.copy_(made)
        st["et"], st["cache"] = et, cache
        if case["kind"] == "attention":
            st["mask"] = {"causal": et.MASK_CAUSAL, "none": et.MASK_NONE}[case["mask"]]
    else:
        st["arrays"] = arrays
    return st


# ---- plain form ---------------------------------------------------------------------------

def _nibbles(b):
    """[..., n] bytes -> [..., 2 n] codes, the low half of a byte first."""
    return torch.stack([b & 15, b >> 4], dim=-1).flatten(-2)


def _k_codes(rows, ng):
    """[..., 16 ng] bytes of K rows -> [..., 32 ng] codes in feature order."""
    lead = rows.shape[:-1]
    n = _nibbles(rows).view(*lead, 4, ng, 8)[..., NIBBLE]
    return n.transpose(-3, -2).reshape(*lead, 32 * ng)


def _v_codes(rows, ng):
    lead = rows.shape[:-1]
    return _nibbles(rows).view(*lead, 8, ng, 4).transpose(-3, -2).reshape(*lead, 32 * ng)


def _values(codes, params):
    s, m = params.to(F32).unbind(-1)
    group = codes.shape[-1] // s.shape[-1]
    c = codes.to(F32).view(*codes.shape[:-1], -1, group)
    return (c * s[..., None] + m[..., None]).view(codes.shape)


def _gather(st, case, pos):
    """Cached K and V in fp32 at positions pos[batch, n]."""
    page, ng = case["page"], _groups(case)
    at = torch.gather(st["table"].long(), 1, pos // page)
    kc, kp, vc, vp = (a[at, :, pos % page] for a in st["arrays"])
    return (_values(_k_codes(kc, ng), kp)[..., : case["dh_qk"]], _values(_v_codes(vc, ng), vp)[..., : case["dh_v"]])


def _attention(st):
    case = st["case"]
    batch, seq, heads, kv = case["batch"], case["seq"], case["heads"], case["kv"]
    pos = torch.arange(case["len"], device="cuda")
    k, v = _gather(st, case, pos.expand(batch, -1))
    q = st["q"].to(F32).view(batch, seq, kv, heads // kv, case["dh_qk"]).permute(0, 2, 3, 1, 4)
    q = q.reshape(batch, kv, heads // kv * seq, case["dh_qk"])
    s = torch.matmul(q, k.permute(0, 2, 3, 1)).view(batch, kv, heads // kv, seq, -1) / math.sqrt(case["dh_qk"])
    last = st["kv_len"].long()[:, None] - 1
    if case["mask"] == "causal":
        last = last - (seq - 1) + torch.arange(seq, device="cuda")
    seen = pos <= last[..., None]
    s = torch.where(seen[:, None, None], s, MASKED)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == MASKED, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = (p / torch.where(total > 0, total, 1.0)).view(batch, kv, -1, p.shape[-1])
    z = torch.matmul(p, v.permute(0, 2, 1, 3)).view(batch, kv, heads // kv, seq, -1)
    return z.permute(0, 3, 1, 2, 4).reshape(batch * seq, -1).to(F16)


def _quantise(x, ng):
    """[..., d] fp16 -> codes [..., 32 ng] and params [..., ng, 2]; features past d stay out of it."""
    lead, d = x.shape[:-1], x.shape[-1]
    wide = torch.nn.functional.pad(x, (0, 32 * ng - d))
    valid = (torch.arange(32 * ng, device=x.device) < d).view(ng, 32)
    x32 = wide.to(F32).view(*lead, ng, 32)
    top, low = torch.where(valid, x32, MASKED).amax(-1), torch.where(valid, x32, -MASKED).amin(-1)
    some = valid.any(-1)
    top, low = torch.where(some, top, 0.0), torch.where(some, low, 0.0)
    s = ((top - low) / 15).to(F16)
    # (the quotient in 64 bits: 32 would round values next to a border between two codes onto it)
    t = (x32.to(F64) - low.to(F64)[..., None]) / torch.where(s == 0, 1.0, s.to(F64))[..., None]
    c = torch.where(valid & (s != 0)[..., None], torch.round(t).clamp(0, 15), 0.0).to(torch.uint8)
    return c.view(*lead, 32 * ng), torch.stack([s, low.to(F16)], dim=-1)


def _bytes(nibbles):
    low, high = nibbles.unflatten(-1, (-1, 2)).unbind(-1)
    return low | (high << 4)


def _k_rows(codes, ng):
    place = sorted(range(8), key=NIBBLE.__getitem__)  # feature at each nibble
    n = codes.view(*codes.shape[:-1], ng, 4, 8)[..., place].transpose(-3, -2)
    return _bytes(n.reshape(codes.shape))


def _v_rows(codes, ng):
    n = codes.view(*codes.shape[:-1], ng, 8, 4).transpose(-3, -2)
    return _bytes(n.reshape(codes.shape))


def _positions(st, case):
    return st["start"].long()[:, None] + torch.arange(case["seq"], device="cuda")


def _read(st):
    case = st["case"]
    k, v = _gather(st, case, _positions(st, case))
    rows = case["batch"] * case["seq"]
    return k.to(F16).reshape(rows, -1), v.to(F16).reshape(rows, -1)


def _write(st):
    case, ng = st["case"], _groups(st["case"])
    batch, seq, kv, page = case["batch"], case["seq"], case["kv"], case["page"]
    kc, kp = _quantise(st["k"].view(batch, seq, kv, -1), ng)
    vc, vp = _quantise(st["v"].view(batch, seq, kv, -1), ng)
    pos = _positions(st, case)
    at = torch.gather(st["table"].long(), 1, pos // page)
    a = st["arrays"]
    a[0][at, :, pos % page], a[1][at, :, pos % page] = _k_rows(kc, ng), kp
    a[2][at, :, pos % page], a[3][at, :, pos % page] = _v_rows(vc, ng), vp


def _linear(st):
    case = st["case"]
    inn, out = case["in"], case["out"]
    nb = st["codes"].shape[1]
    # [panel, block, half, row, j, word, nibble] -> [panel, half, row, block, word, j, feature]
    n = _nibbles(st["codes"].view(out // 16, nb, 2, 8, 4, 4, 4))[..., NIBBLE]
    n = n.permute(0, 2, 3, 1, 5, 4, 6).reshape(out, nb * 128)
    w = _values(n, st["params"].transpose(1, 2).reshape(out, -1, 2))[:, :inn]
    y = st["x"].to(F32) @ w.T
    if st["bias"] is not None:
        y = y + st["bias"].to(F32)
    if case["act"] == "relu":
        y = torch.relu(y)
    return y.to(F16)


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        et = state["et"]
        if kind == "linear":
            return et.linear_w4(state["x"], state["weight"], state["bias"], state["act"])
        if kind == "attention":
            return et.attention_kv4(state["cache"], state["q"], state["table"], state["kv_len"], case["batch"],
                                    case["seq"], case["heads"], max_len=case["len"], mask_kind=state["mask"])
        if kind == "cache":
            et.kv4_write(state["cache"], state["k"], state["v"], state["table"], state["start"], case["batch"],
                         case["seq"])
        return et.kv4_read(state["cache"], state["table"], case["batch"], case["seq"], start=state["start"])
    if kind == "linear":
        return _linear(state)
    if kind == "attention":
        return _attention(state)
    if kind == "cache":
        _write(state)
    return _read(state)


def work(case):
    if case["kind"] == "linear":
        T, inn, out = case["T"], case["in"], case["out"]
        return {"bytes": inn * out * (0.5 + 4.0 / case["group"]) + 2 * T * (inn + out) + (2 * out if case["bias"] else 0),
                "flops": 2.0 * T * inn * out}
    width = case["dh_qk"] + case["dh_v"]
    if case["kind"] == "attention":
        keys, seq = sum(_lengths(case)), case["seq"]
        scores = seq * keys
        if case["mask"] == "causal":
            scores -= case["batch"] * seq * (seq - 1) // 2
        return {"bytes": keys * case["kv"] * width * 0.625 + 2 * case["batch"] * seq * case["heads"] * width
                + 4 * case["batch"] * (1 + -(-case["len"] // case["page"])),
                "flops": 2.0 * case["heads"] * scores * width}
    values = case["batch"] * case["seq"] * case["kv"] * width
    once = 2.0 + 0.625  # the fp16 value and the 4-bit one
    return {"bytes": values * once * (2 if case["kind"] == "cache" else 1),
            "flops": values * (10.0 if case["kind"] == "cache" else 2.0)}


# ---- the definition in 64 bits ---------------------------------------------------------------

def _word_codes(words, order):
    """32-bit words -> codes of the features in `order`, one at a time by shifts."""
    w = words.to(torch.int64) & 0xFFFFFFFF
    return torch.stack([(w >> (4 * p)) & 15 for p in order], dim=-1).to(F64)


def _k64(codes, params, d):
    ng = params.shape[-2]
    w = _word_codes(codes.contiguous().view(torch.int32), [0, 4, 1, 5, 2, 6, 3, 7])  # [..., 4 ng, 8]
    p = params.to(F64)
    out = torch.empty((*codes.shape[:-1], 32 * ng), dtype=F64, device=codes.device)
    for g in range(ng):
        for j in range(4):
            out[..., 32 * g + 8 * j: 32 * g + 8 * j + 8] = w[..., j * ng + g, :] * p[..., g, 0, None] + p[..., g, 1, None]
    return out[..., :d]


def _v64(codes, params, d):
    ng = params.shape[-2]
    b = codes.to(torch.int64)
    p = params.to(F64)
    out = torch.empty((*codes.shape[:-1], 32 * ng), dtype=F64, device=codes.device)
    for g in range(ng):
        for i in range(8):
            unit = b[..., 2 * (i * ng + g)] + 256 * b[..., 2 * (i * ng + g) + 1]
            for f in range(4):
                out[..., 32 * g + 4 * i + f] = ((unit >> (4 * f)) & 15).to(F64) * p[..., g, 0] + p[..., g, 1]
    return out[..., :d]


def _rounded64(x):
    """[..., n] fp16 -> the values that 4-bit groups of 32 stand for, in 64 bits."""
    d = x.shape[-1]
    out = torch.empty(x.shape, dtype=F64, device=x.device)
    for lo in range(0, d, 32):
        v = x[..., lo: lo + 32].to(F64)
        low, high = v.min(-1, keepdim=True).values, v.max(-1, keepdim=True).values
        s = ((high.to(F32) - low.to(F32)) / 15).to(F16).to(F64)
        c = torch.where(s > 0, torch.round((v - low) / s.clamp(min=2.0 ** -24)), 0.0).clamp(0, 15)
        out[..., lo: lo + 32] = c * s + low
    return out


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "linear":
        inn, out, group = case["in"], case["out"], case["group"]
        words = st["codes"].view(torch.int32).view(out // 16, -1, 2, 8, 4, 4)
        w = torch.empty((out // 16, 2, 8, words.shape[1] * 128), dtype=F64, device="cuda")
        p = st["params"].to(F64).transpose(1, 2).reshape(out // 16, 2, 8, -1, 2)
        for j in range(4):
            for n in range(4):
                c = _word_codes(words[..., j, n], [0, 4, 1, 5, 2, 6, 3, 7]).permute(0, 2, 3, 1, 4)
                at = torch.arange(words.shape[1], device="cuda") * 128 + 32 * n + 8 * j
                s = p[:, :, :, at // group]
                w[..., at[:, None] + torch.arange(8, device="cuda")] = c * s[..., 0, None] + s[..., 1, None]
        y = st["x"].to(F64) @ w.view(out, -1)[:, :inn].T
        y = y + st["bias"].to(F64) if st["bias"] is not None else y
        return y.clamp(min=0) if case["act"] == "relu" else y
    batch, seq, kv, page = case["batch"], case["seq"], case["kv"], case["page"]
    rows = batch * seq
    if case["kind"] == "cache":
        return (_rounded64(st["k"].view(rows, kv, -1)).view(rows, -1), _rounded64(st["v"].view(rows, kv, -1)).view(rows, -1))
    kc, kp, vc, vp = st["arrays"]
    zs, ks, vs = [], [], []
    for b in range(batch):
        first = case.get("start", 0)
        last = _lengths(case)[b] if case["kind"] == "attention" else first + seq
        at = st["table"][b].long()
        pos = torch.arange(first, last, device="cuda")
        take = lambda a: a[at[pos // page], :, pos % page]  # noqa: E731
        k = _k64(take(kc), take(kp), case["dh_qk"])
        v = _v64(take(vc), take(vp), case["dh_v"])
        if case["kind"] == "read":
            ks.append(k.reshape(seq, -1))
            vs.append(v.reshape(seq, -1))
            continue
        q = st["q"].to(F64).view(rows, -1, case["dh_qk"])[b * seq: (b + 1) * seq]
        for h in range(case["heads"]):
            of = h // (case["heads"] // kv)
            s = (q[:, h] @ k[:, of].T) * case["dh_qk"] ** -0.5
            if case["mask"] == "causal":
                limit = last - seq + torch.arange(seq, device="cuda")
                s = s.masked_fill(pos[None] > limit[:, None], MASKED)
            zs.append(torch.softmax(s, -1) @ v[:, of])
    if case["kind"] == "read":
        return torch.cat(ks), torch.cat(vs)
    return torch.stack(zs).view(batch, case["heads"], seq, -1).transpose(1, 2).reshape(rows, -1)
