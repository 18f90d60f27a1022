"""Performance cases of the transformer operators in the int8 numerics of the library: a paged int8 cache of keys and values
(append, read, attention over it) and int8 products grouped by expert.

A case is a dict of plain values. Its "kind" is one of

  append   new keys and values into the cache (KvCache.append), and the tokens of every block that it touched read back
           (KvCache.read)
  read     the tokens of the cache as floats (KvCache.read)
  attend   attention of tokens that are in the cache already (KvCache.attend)
  step     the two calls of a decoding step: append, then attend
  linear   int8 products of rows sorted by expert, with a scale for each row found on the way in (Linear.forward)

The plain forms below are elementary torch operations on the same inputs, in 32 bits but for the quotients that are rounded to
codes. `exact` computes the operators from their definition in 64 bits.
"""
import math
import random

import torch

own = False

BLOCK = 64  # tokens that share a scale, and a page of the cache

# What a drawn case may cost at most: the listed ones' largest.
MOST_BYTES = 4.8e8
MOST_FLOPS = {"attend": 8.0e11, "step": 8.0e11, "linear": 2.6e11}


def _cache(name=None, *, kind, seqs, heads, dim, old, new, group=1, ragged=0, cap=0.0, window=0, slopes=False, causal=True):
    """`old` tokens are in the cache before, `new` ones come; ragged != 0: lengths up to these, drawn by that number."""
    c = dict(kind=kind, seqs=seqs, heads=heads, dim=dim, old=old, new=new, ragged=ragged)
    if kind in ("attend", "step"):
        c.update(group=group, cap=cap, window=window, slopes=slopes, causal=causal)
    return dict(c, name=name) if name else c


def _linear(name=None, *, experts, tokens, top, k, n, gated=False, act="", bias=True, ragged=1):
    c = dict(kind="linear", experts=experts, tokens=tokens, top=top, k=k, n=n, gated=gated, act=act, bias=bias, ragged=ragged)
    return dict(c, name=name) if name else c


def listed():
    return [
        # the cache's half of a decoding step of a serving batch: one token each, blocks partly filled (latency)
        _cache("append_token", kind="append", seqs=48, heads=8, dim=128, old=900, new=1, ragged=3),
        # prompts of a batch go into the cache, behind what an earlier part of them left there
        _cache("append_prompts", kind="append", seqs=12, heads=8, dim=128, old=300, new=2000, ragged=5),
        # a batch's caches as floats, for a transfer or an inspection
        _cache("read_batch", kind="read", seqs=16, heads=8, dim=128, old=0, new=2048, ragged=7),
        # a small model answers one user: one token, a short cache (latency)
        _cache("attend_one", kind="attend", seqs=1, heads=4, group=2, dim=64, old=520, new=1),
        # one user, one token, a very long cache: few rows, a long axis
        _cache("attend_long", kind="attend", seqs=1, heads=4, group=7, dim=128, old=200000, new=1),
        # prompts of a batch in a model with capped scores, distance slopes and a window
        _cache("attend_prompts", kind="attend", seqs=6, heads=16, dim=64, old=0, new=1900, ragged=11, cap=30.0, window=512, slopes=True),
        # a part of a long prompt against what is in the cache: the most operations of the range
        _cache("attend_chunk", kind="attend", seqs=1, heads=8, group=4, dim=128, old=10000, new=4096),
        # a decoding step of a full serving batch: the most bytes of the range
        _cache("step_batch", kind="step", seqs=64, heads=8, group=4, dim=128, old=7000, new=1, ragged=13),
        # one row through one projection (latency)
        _linear("linear_row", experts=1, tokens=1, top=1, k=2048, n=2048, bias=False),
        # a decoding step's rows on experts with a gate, sizes that fill no tile: the weights are the traffic
        _linear("linear_experts_few", experts=16, tokens=24, top=2, k=1032, n=1384, gated=True),
        # a prompt's rows on experts, the product behind the gate
        _linear("linear_experts", experts=8, tokens=4096, top=2, k=2816, n=2048, bias=True),
        # a projection of a prompt's rows with an activation: the largest product
        _linear("linear_projection", experts=1, tokens=8192, top=1, k=4096, n=4000, act="Relu"),
    ]


# ------------------------------------------------------------------------------------------------------
# drawn cases
# ------------------------------------------------------------------------------------------------------

def _log_int(rng, lo, hi):
    """A whole number whose logarithm is spread evenly over [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _smaller(case):
    for key, least in (("seqs", 1), ("tokens", 1), ("old", 0), ("new", 1), ("heads", 1), ("n", 16), ("k", 16), ("experts", 1)):
        if case.get(key, least) > max(least, 64 if key in ("old", "new") else least):
            case = dict(case, **{key: max(least, int(case[key] * 0.75))})
            if "top" in case:
                case["top"] = min(case["top"], case["experts"])
            return case
    return case


def draw(rng):
    what = rng.random()
    ragged = rng.randint(1, 1 << 30)
    if what < 0.6:
        heads, dim = _log_int(rng, 1, 16), rng.choice((64, 64, 128, 128, 128, 128, 32, 80, 96, 256))
        seqs = _log_int(rng, 1, 64)
        common = dict(seqs=seqs, heads=heads, dim=dim, ragged=rng.choice((0, ragged, ragged)))
        if what < 0.12:
            one = rng.random() < 0.5
            case = _cache(kind="append", old=_log_int(rng, 1, 4000) - 1, new=1 if one else _log_int(rng, 2, 4000), **common)
        elif what < 0.18:
            case = _cache(kind="read", old=0, new=_log_int(rng, 1, 4000), **common)
        else:
            more = dict(group=rng.choice((1, 1, 2, 4, 4, 5, 8)), cap=rng.choice((0.0, 0.0, 0.0, 20.0, 50.0)),
                        window=rng.choice((0, 0, 0, _log_int(rng, 16, 4000))), slopes=rng.random() < 0.2, **common)
            if what < 0.30:
                case = _cache(kind="step", old=_log_int(rng, 1, 16000) - 1, new=1, **more)
            elif what < 0.40:
                more.update(seqs=_log_int(rng, 1, 4))
                case = _cache(kind="attend", old=_log_int(rng, 1, 200000) - 1, new=rng.choice((1, 1, 2, 4)), **more)
            else:
                more.update(seqs=_log_int(rng, 1, 16))
                case = _cache(kind="attend", old=rng.choice((0, _log_int(rng, 1, 10000))), new=_log_int(rng, 2, 4000),
                              causal=rng.random() < 0.85, **more)
    else:
        experts = rng.choice((1, 1, 1, _log_int(rng, 2, 64)))
        case = _linear(experts=experts, tokens=_log_int(rng, 1, 8192), top=min(experts, rng.choice((1, 2, 2, 4))),
                       k=_log_int(rng, 64, 8192), n=_log_int(rng, 16, 8192), gated=rng.random() < 0.3, bias=rng.random() < 0.5,
                       ragged=ragged)
        if not case["gated"]:
            case["act"] = rng.choice(("", "", "", "Relu", "LRelu", "Relu6", "Sigmoid"))
        if case["k"] > 256 and rng.random() < 0.7:  # most layers' sizes are whole multiples
            case.update(k=case["k"] // 64 * 64, n=max(16, case["n"] // 16 * 16))
    while True:
        w = work(case)
        if w["bytes"] <= MOST_BYTES and w["flops"] <= MOST_FLOPS.get(case["kind"], 1e15):
            return case
        case = _smaller(case)


# ------------------------------------------------------------------------------------------------------
# lengths and routes: from the case alone
# ------------------------------------------------------------------------------------------------------

def _lengths(case):
    """(tokens that are there before, tokens that come) for each sequence; the first has the most of both."""
    if not case["ragged"]:
        return [(case["old"], case["new"])] * case["seqs"]
    rng = random.Random(case["ragged"])
    rest = [(rng.randint(0, case["old"]), rng.randint(1, case["new"])) for _ in range(case["seqs"] - 1)]
    return [(case["old"], case["new"])] + rest


def _route(case):
    """The row of x that each of the sorted rows is, and where each expert's rows start. Some experts are preferred."""
    e, t, top = case["experts"], case["tokens"], case["top"]
    if e == 1:
        return None, [0, t]
    rng = random.Random(case["ragged"])
    likes = [rng.random() + 0.2 for _ in range(e)]
    rows = [[] for _ in range(e)]
    for i in range(t):
        left = list(range(e))
        for _ in range(top):
            one = rng.choices(left, [likes[j] for j in left])[0]
            left.remove(one)
            rows[one].append(i)
    starts = [0]
    for r in rows:
        starts.append(starts[-1] + len(r))
    return [i for r in rows for i in r], starts


def _seen(case, old, new):
    """Query-key pairs of a sequence, and the cache's tokens that any of them reads."""
    total, window = old + new, case["window"]
    pairs = 0
    for r in range(new):
        p = old + r
        last = p if case["causal"] else total - 1
        first = max(0, p - window + 1) if window else 0
        pairs += last - first + 1
    return pairs, total - (max(0, old - window + 1) if window else 0)


def work(case):
    if case["kind"] == "linear":
        index, starts = _route(case)
        rows, n = starts[-1], case["n"] * (2 if case["gated"] else 1)
        used = sum(b > a for a, b in zip(starts, starts[1:]))
        return {"bytes": used * n * (case["k"] + 4 + 4 * case["bias"]) + 4 * case["tokens"] * case["k"] + 4 * rows * case["n"],
                "flops": 2 * rows * n * case["k"]}
    token = 2 * case["heads"] * case["dim"]  # key and value of a token, in elements
    lengths = _lengths(case)
    news = sum(n for _, n in lengths)
    nbytes = flops = 0
    if case["kind"] in ("append", "step"):
        nbytes += news * token * 5 + sum(o % BLOCK for o, _ in lengths) * token
    if case["kind"] == "append":
        nbytes += sum(n + o % BLOCK for o, n in lengths) * token * 5
    if case["kind"] == "read":
        nbytes += news * token * 5
    if case["kind"] in ("attend", "step"):
        for o, n in lengths:
            pairs, tokens = _seen(case, o, n)
            flops += 4 * case["dim"] * case["heads"] * case["group"] * pairs
            nbytes += tokens * token + -(-tokens // BLOCK) * 8 * case["heads"] + 4 * n * token * case["group"]
    return {"bytes": nbytes, "flops": flops}


# ------------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------------

_library = []


def _lib():
    if not _library:
        from tensor_amd import capi
        _library.append(capi.Library(0))
    return _library[0]


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _cache_inputs(case, seed):
    """Tokens before and new ones, queries, slopes, and the page table: pages in no order, as an allocator hands them out."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    lengths = _lengths(case)
    heads, dim = case["heads"], case["dim"]
    olds, news = sum(o for o, _ in lengths), sum(n for _, n in lengths)
    # a few channels of the keys are far larger than the others, as in trained models
    channel = 1 + 5 * (torch.rand((heads, dim), generator=gen, device="cuda") > 0.97)
    i = dict(lengths=lengths, old_k=_normal(gen, olds, heads, dim) * channel, old_v=_normal(gen, olds, heads, dim),
             new_k=_normal(gen, news, heads, dim) * channel, new_v=_normal(gen, news, heads, dim))
    if "group" in case:
        i["q"] = _normal(gen, news, heads * case["group"], dim) * 1.5
        i["slopes"] = torch.exp2(-8.0 * torch.arange(1, heads * case["group"] + 1, device="cuda") / (heads * case["group"])).float() \
            if case["slopes"] else None
    need = [-(-(o + n) // BLOCK) for o, n in lengths]
    order = torch.randperm(sum(need) + 3, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros((len(need), max(need)), dtype=torch.int32, device="cuda")
    at = 0
    for s, k in enumerate(need):
        table[s, :k] = order[at:at + k]
        at += k
    i.update(table=table, pages=sum(need) + 3)
    return i


def _batch(counts, lengths):
    """starts and lengths of a batch, on the GPU, and its rows."""
    starts = [0]
    for c in counts:
        starts.append(starts[-1] + c)
    return (torch.tensor(starts, dtype=torch.int32, device="cuda"), torch.tensor(lengths, dtype=torch.int32, device="cuda"), starts[-1])


def _linear_inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    e, k, n = case["experts"], case["k"], case["n"] * (2 if case["gated"] else 1)
    index, starts = _route(case)
    # rows of different size, some channels far larger than the others
    x = _normal(gen, case["tokens"], k) * torch.exp(0.5 * _normal(gen, case["tokens"], 1)) * \
        (1 + 4 * (torch.rand((1, k), generator=gen, device="cuda") > 0.99))
    w = (_normal(gen, e, n, k) * 36).round_().clamp_(-127, 127).to(torch.int8)
    scale = (0.5 + torch.rand((e, n), generator=gen, device="cuda")) / (36 * math.sqrt(k))
    return dict(x=x, w=w, scale=scale, bias=0.1 * _normal(gen, e, n) if case["bias"] else None,
                starts=torch.tensor(starts, dtype=torch.int32, device="cuda"), bounds=starts,
                index=None if index is None else torch.tensor(index, dtype=torch.int32, device="cuda"))


def prepare(case, seed):
    s = dict(case=case)
    if case["kind"] == "linear":
        i = _linear_inputs(case, seed)
        s.update(x=i["x"], starts=i["starts"], index=i["index"])
        if own:
            from tensor_amd import capi
            s["layer"] = _lib().linear(weight=i["w"].cpu().numpy(), scale=i["scale"].cpu().numpy(), gated=case["gated"],
                                       bias=None if i["bias"] is None else i["bias"].cpu().numpy(), act=capi.ACT[case["act"]],
                                       act_p0=0.1 if case["act"] == "LRelu" else 0.0)
        else:
            s.update(w=i["w"], scale=i["scale"], bias=i["bias"], bounds=i["bounds"])
        return s
    i = _cache_inputs(case, seed)
    lengths = i["lengths"]
    before, batch = _batch([o for o, _ in lengths], [o for o, _ in lengths]), _batch([n for _, n in lengths], [o + n for o, n in lengths])
    tail = _batch([n + o % BLOCK for o, n in lengths], [o + n for o, n in lengths])
    s.update(k=i["new_k"], v=i["new_v"], q=i.get("q"), slopes=i.get("slopes"))
    if own:
        cache = _lib().kv_cache(i["pages"], case["heads"], case["dim"])
        made = [_lib().kv_batch(b[0], b[1], i["table"], b[2]) for b in (before, batch, tail)]
        if before[2]:
            cache.append(made[0], i["old_k"], i["old_v"])
        if case["kind"] in ("read", "attend"):
            cache.append(made[1], i["new_k"], i["new_v"])
        s.update(cache=cache, batch=made[1], tail=made[2])
    else:
        shape = (i["pages"], BLOCK, case["heads"], case["dim"])
        cache = dict(table=i["table"])
        for part in "kv":
            cache[part] = torch.zeros(shape, dtype=torch.int8, device="cuda")
            cache[part + "s"] = torch.zeros((i["pages"], case["heads"]), device="cuda")
        if before[2]:
            _append(cache, before, i["old_k"], i["old_v"])
        if case["kind"] in ("read", "attend"):
            _append(cache, batch, i["new_k"], i["new_v"])
        s.update(cache=cache, batch=batch, tail=tail, lengths=lengths)
    return s


# ------------------------------------------------------------------------------------------------------
# the plain forms
# ------------------------------------------------------------------------------------------------------

def _codes(x, s):
    """x / s rounded half away from zero, at most 127; 0 where the scale is."""
    q = torch.where(s > 0, x.double() / s.double(), 0.0)
    return (torch.sign(q) * torch.floor(q.abs() + 0.5)).clamp_(-127, 127).to(torch.int8)


def _scale_of(most):
    s = (most.double() / 127).float()
    return torch.where(s < 2.0 ** -100, 0.0, s)


def _rows(batch):
    """Sequence and position of every row of a batch."""
    starts, lengths, total = batch
    counts = starts[1:] - starts[:-1]
    seq = torch.repeat_interleave(torch.arange(len(lengths), device="cuda"), counts, output_size=total)
    pos = torch.arange(total, device="cuda") - starts[:-1][seq] + (lengths - counts)[seq]
    return seq, pos


def _append(cache, batch, keys, values):
    starts, lengths, total = batch
    seq, pos = _rows(batch)
    page = cache["table"][seq, pos // BLOCK].long()
    first = lengths - (starts[1:] - starts[:-1])  # where the new tokens begin
    has = ((first % BLOCK) > 0) & (starts[1:] > starts[:-1])  # blocks with older tokens
    block = cache["table"].gather(1, (first // BLOCK).long().clamp(max=cache["table"].shape[1] - 1)[:, None])[:, 0].long()[has]
    older = torch.arange(BLOCK, device="cuda")[None, :] < (first % BLOCK)[has][:, None]
    touched = torch.zeros(len(cache["k"]), dtype=torch.bool, device="cuda").index_fill_(0, page, True)
    for part, x in (("k", keys), ("v", values)):
        codes, scales = cache[part], cache[part + "s"]
        most = torch.zeros_like(scales).index_reduce_(0, page, x.abs().amax(-1), "amax")
        s = _scale_of(most)
        was = scales[block]
        s[block] = torch.maximum(s[block], was)
        old = codes[block]
        again = _codes(old.double() * was.double()[:, None, :, None], s[block][:, None, :, None])
        codes[block] = torch.where(older[:, :, None, None], again, old)
        scales.copy_(torch.where(touched[:, None], s, scales))
        codes[page, pos % BLOCK] = _codes(x, scales[page][:, :, None])


def _read(cache, batch):
    seq, pos = _rows(batch)
    page, slot = cache["table"][seq, pos // BLOCK].long(), pos % BLOCK
    return tuple(cache[p][page, slot].float() * cache[p + "s"][page][:, :, None] for p in "kv")


def _attend(state):
    case, cache, q = state["case"], state["cache"], state["q"]
    heads, group, dim = case["heads"], case["group"], case["dim"]
    out = torch.empty_like(q)
    at = 0
    for s, (o, n) in enumerate(state["lengths"]):
        total = o + n
        begin = max(0, o - case["window"] + 1) // BLOCK if case["window"] else 0  # blocks that nobody sees are not read
        pages = cache["table"][s, begin:-(-total // BLOCK)].long()
        k, v = (cache[p][pages].float() * cache[p + "s"][pages][:, None, :, None] for p in "kv")
        k, v = (t.reshape(-1, heads, dim)[:total - begin * BLOCK].permute(1, 0, 2).contiguous() for t in (k, v))
        mine = q[at:at + n].reshape(n, heads, group, dim).permute(1, 2, 0, 3).reshape(heads, group * n, dim)
        p = torch.arange(o, total, device="cuda")[:, None]
        j = torch.arange(begin * BLOCK, total, device="cuda")[None, :]
        hidden = torch.zeros((n, total - begin * BLOCK), dtype=torch.bool, device="cuda")
        if case["causal"]:
            hidden |= j > p
        if case["window"]:
            hidden |= j <= p - case["window"]
        t = torch.matmul(mine, k.transpose(1, 2).contiguous()).mul_(1 / math.sqrt(dim)).reshape(heads, group, n, -1)
        if case["cap"]:
            t = torch.tanh(t / case["cap"]).mul_(case["cap"])
        if case["slopes"]:
            t = t - state["slopes"].reshape(heads, group, 1, 1) * (p - j).abs().float()
        t = t.masked_fill_(hidden, -math.inf)
        t = torch.exp(t - t.amax(-1, keepdim=True))
        total_weight = t.sum(-1, keepdim=True)
        r = torch.matmul(t.reshape(heads, group * n, -1), v).reshape(heads, group, n, dim) / total_weight
        out[at:at + n] = r.permute(2, 0, 1, 3).reshape(n, heads * group, dim)
        at += n
    return out


def _activate(y, act):
    if act == "Relu":
        return y.clamp(min=0)
    if act == "LRelu":
        return torch.where(y > 0, y, y * 0.1)
    if act == "Relu6":
        return y.clamp(0, 6)
    if act == "Sigmoid":
        return 1 / (1 + torch.exp(-y))
    return y


def _linear_plain(state):
    case, x = state["case"], state["x"]
    xs = _scale_of(x.abs().amax(-1, keepdim=True))
    codes = _codes(x, xs).float()
    if state["index"] is not None:
        codes, xs = codes[state["index"]], xs[state["index"]]
    y = torch.empty((len(codes), case["n"]), device="cuda")
    for e, (a, b) in enumerate(zip(state["bounds"], state["bounds"][1:])):
        if a == b:
            continue
        # the sums are whole numbers below 2^24 in size for such inputs: exact
        z = torch.matmul(codes[a:b], state["w"][e].float().t()) * (xs[a:b] * state["scale"][e])
        if state["bias"] is not None:
            z = z + state["bias"][e]
        if case["gated"]:
            gate, up = z[:, :case["n"]], z[:, case["n"]:]
            z = gate / (1 + torch.exp(-gate)) * up
        y[a:b] = _activate(z, case["act"])
    return y


def run(state):
    kind = state["case"]["kind"]
    if not own:
        if kind == "linear":
            return _linear_plain(state)
        if kind in ("append", "step"):
            _append(state["cache"], state["batch"], state["k"], state["v"])
        if kind == "append":
            return _read(state["cache"], state["tail"])
        return _read(state["cache"], state["batch"]) if kind == "read" else _attend(state)
    if kind == "linear":
        if state["index"] is None:
            return state["layer"].forward(state["x"])
        return state["layer"].forward(state["x"], starts=state["starts"], index=state["index"])
    cache, batch, case = state["cache"], state["batch"], state["case"]
    if kind in ("append", "step"):
        cache.append(batch, state["k"], state["v"])
    if kind == "append":
        return cache.read(state["tail"])
    if kind == "read":
        return cache.read(batch)
    return cache.attend(batch, state["q"], cap=case["cap"], window=case["window"], slopes=state["slopes"], causal=case["causal"])


# ------------------------------------------------------------------------------------------------------
# the definition, in 64 bits
# ------------------------------------------------------------------------------------------------------

def _nearest(q):
    """Half away from zero, of 64-bit quotients."""
    return torch.where(q < 0, -torch.floor(0.5 - q), torch.floor(0.5 + q)).clamp(-127, 127)


def _stored(old, new):
    """What the cache stands for after `old` and then `new` tokens of one sequence went in: [tokens, heads, dim] in 64 bits."""
    o, total = len(old), len(old) + len(new)
    blocks = -(-total // BLOCK)
    earlier, later = (torch.zeros((blocks * BLOCK,) + new.shape[1:], dtype=torch.float64, device=new.device) for _ in range(2))
    earlier[:o], later[o:total] = old.double(), new.double()
    earlier, later = (t.reshape(blocks, BLOCK, *new.shape[1:]) for t in (earlier, later))
    s0, s1 = ((t.abs().amax((1, 3), keepdim=True) / 127).float().double() for t in (earlier, later))  # a scale is a 32-bit number
    s = torch.maximum(s0, s1)
    c = _nearest(earlier / s0.clamp(min=1e-300))
    c = torch.where(s > s0, _nearest(c * s0 / s.clamp(min=1e-300)), c)
    is_new = (torch.arange(blocks * BLOCK, device=new.device) >= o).reshape(blocks, BLOCK, 1, 1)
    c = torch.where(is_new, _nearest(later / s.clamp(min=1e-300)), c)
    return (c * s).reshape(blocks * BLOCK, *new.shape[1:])[:total]


def exact(case, seed):
    if case["kind"] == "linear":
        i = _linear_inputs(case, seed)
        x = i["x"].double()
        xs = (x.abs().amax(1) / 127).float().double()
        c = _nearest(x / xs[:, None].clamp(min=1e-300))
        rows = torch.arange(len(x), device="cuda") if i["index"] is None else i["index"].long()
        out = []
        for e in range(case["experts"]):
            r = rows[i["bounds"][e]:i["bounds"][e + 1]]
            z = (c[r] @ i["w"][e].double().T) * xs[r][:, None] * i["scale"][e].double()
            if i["bias"] is not None:
                z += i["bias"][e].double()
            if case["gated"]:
                z = z[:, :case["n"]] * torch.sigmoid(z[:, :case["n"]]) * z[:, case["n"]:]
            elif case["act"] == "Sigmoid":
                z = torch.sigmoid(z)
            elif case["act"] == "Relu6":
                z = torch.minimum(torch.relu(z), torch.full_like(z, 6.0))
            elif case["act"] == "Relu":
                z = torch.relu(z)
            elif case["act"] == "LRelu":
                z = torch.relu(z) - float(torch.tensor(0.1, dtype=torch.float32)) * torch.relu(-z)
            out.append(z)
        return torch.cat(out)
    i = _cache_inputs(case, seed)
    heads, dim, group = case["heads"], case["dim"], case.get("group", 1)
    ks, vs, outs = [], [], []
    oa = na = 0
    for o, n in i["lengths"]:
        empty = i["old_k"][:0]
        if case["kind"] == "read":
            k, v = (_stored(empty, i["new_" + p][na:na + n]) for p in "kv")
            ks.append(k), vs.append(v)
        else:
            k, v = (_stored(i["old_" + p][oa:oa + o], i["new_" + p][na:na + n]) for p in "kv")
            if case["kind"] == "append":
                ks.append(k[o - o % BLOCK:]), vs.append(v[o - o % BLOCK:])
            else:
                one = torch.empty((n, heads * group, dim), dtype=torch.float64, device="cuda")
                where = torch.arange(o + n, device="cuda")
                away = where[o:, None] - where[None, :]
                sees = torch.ones_like(away, dtype=torch.bool)
                if case["causal"]:
                    sees &= away >= 0
                if case["window"]:
                    sees &= away < case["window"]
                for h in range(heads * group):
                    t = (i["q"][na:na + n, h].double() @ k[:, h // group].T) / math.sqrt(dim)
                    if case["cap"]:
                        t = case["cap"] * torch.tanh(t / case["cap"])
                    if case["slopes"]:
                        t = t - i["slopes"][h].double() * away.abs()
                    t = torch.where(sees, t, -math.inf)
                    one[:, h] = torch.softmax(t, 1) @ v[:, h // group]
                outs.append(one)
        oa, na = oa + o, na + n
    return torch.cat(outs) if outs else (torch.cat(ks), torch.cat(vs))
