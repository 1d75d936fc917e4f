"""Serving from a 4-bit paged key/value cache with drafted tokens, as measurable
cases.

Four operators of torch.ops.cbq (cbq_ops.load()), each with its plain form in
elementary torch operations:

- "append": paged_append_q4, the head norm and rotation of new tokens' queries
  and keys, and the keys and values into 4-bit pages; and paged_read_q4 of the
  same rows, what the cache holds of them now;
- "read": paged_read_q4, rows of the cache as values;
- "decode": prefix_attention_decode_q4, the newest tokens of each sequence of a
  batch (one, or one and its drafts) over a cache of 4 bits;
- "verify": verify_drafts, drafted tokens against the target's probabilities
  from given random numbers, and the token behind those that are kept.

Pages are [n_pages, n_kv, page, hd / 2] bytes and [n_pages, n_kv, page, hd / 64,
2] bf16 numbers (scale s, mid m): 64 neighbouring values of a row are m + s (c -
7.5).  A row's codes lie four of each of its groups side by side (values 0..3, 64..67,
.. 4..7, 68..71, ..), the first of two in a byte's low half.  Head layouts and the
vocabulary are those of the two decoder configurations of
codebook-quantization_amd/synthetic.py (32 and 16 query heads on 8 kv heads of
128, 151936 tokens) and generic ones of the other head sizes.
"""
import math
import os
import random
import sys

import torch

own = False                  # True: run() calls the framework's operators

EPS = 1.0e-6
THETA = 1.0e6
GROUP = 64                   # values that share a scale and a mid
_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}
_STORED = 0.5 + 4 / GROUP    # bytes of a value in the cache


def _append(name, dtype, batch, past, lo, hi, n_q, n_kv, hd, page, rot=None, norm=True):
    """batch runs of lo..hi new tokens each, behind `past` cached ones."""
    return dict(name=name, op="append", dtype=dtype, batch=batch, past=past, lo=lo, hi=hi, n_q=n_q,
                n_kv=n_kv, hd=hd, page=page, rot=rot or hd, norm=norm)


def _read(name, dtype, rows, n_kv, hd, page):
    """`rows` cached tokens in order."""
    return dict(name=name, op="read", dtype=dtype, rows=rows, n_kv=n_kv, hd=hd, page=page)


def _decode(name, dtype, batch, tokens, prefix, lo, hi, n_q, n_kv, hd, page):
    """`tokens` newest tokens of batch sequences of lo..hi own keys each (theirs
    included) behind `prefix` shared ones."""
    return dict(name=name, op="decode", dtype=dtype, batch=batch, tokens=tokens, prefix=prefix,
                lo=lo, hi=hi, n_q=n_q, n_kv=n_kv, hd=hd, page=page)


def _verify(name, dtype, batch, drafts, vocab, spread, given=True):
    """batch sequences with `drafts` drafted tokens each; spread: how far the
    draft's logits are from the target's; given: whether the draft has
    probabilities (or names its tokens for certain)."""
    return dict(name=name, op="verify", dtype=dtype, batch=batch, drafts=drafts, vocab=vocab,
                spread=spread, given=given)


def listed():
    return [
        # one token of one sequence of the fp32 decoder, 8B head layout: latency
        _append("append-1-f32", "f32", 1, 383, 1, 1, 32, 8, 128, 16),
        # a step of a batch with four drafts a sequence, 1.7B head layout, half of
        # each head rotated, no norm
        _append("append-48x5-f16", "f16", 48, 200, 5, 5, 16, 8, 128, 32, rot=64, norm=False),
        # a scheduler's pass over many prompts at once, 8B head layout
        _append("append-prompts-bf16", "bf16", 24, 0, 40, 1000, 32, 8, 128, 64),
        # the fp32 decoder's 128-token prompt and 256 tokens behind it, looked up
        _read("read-384-f32", "f32", 384, 8, 128, 16),
        # a long shared document, for the attention of new prompts behind it
        _read("read-30011-bf16", "bf16", 30011, 8, 128, 64),
        # one sequence of the fp32 decoder, no prefix: latency
        _decode("decode-1x384-f32", "f32", 1, 1, 0, 384, 384, 32, 8, 128, 16),
        # a batch behind a system prompt, three drafts a sequence, 1.7B head layout
        _decode("decode-16x4-bf16-prefix1000", "bf16", 16, 4, 1000, 100, 400, 16, 8, 128, 32),
        # heads of 64 in groups of twelve, very uneven lengths, two drafts, fp16
        _decode("decode-33x3-f16-prefix5000", "f16", 33, 3, 5000, 3, 2900, 24, 2, 64, 128),
        # many questions about one long document, 8B head layout
        _decode("decode-64-bf16-prefix30011", "bf16", 64, 1, 30011, 200, 1500, 32, 8, 128, 64),
        # long conversations, no prefix, 8B head layout: the most bytes
        _decode("decode-24-bf16-long", "bf16", 24, 1, 0, 4000, 32000, 32, 8, 128, 64),
        # four drafts of one sequence: latency
        _verify("verify-1x4-f32", "f32", 1, 4, 151936, 0.7),
        # seven drafts each of a large batch
        _verify("verify-64x7-f32", "f32", 64, 7, 151936, 0.5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges, no larger than its operator's largest."""
    op = rng.choice(["append", "read", "decode", "decode", "verify"])
    every = [work(c) for c in listed() if c["op"] == op]
    most = {k: max(w[k] for w in every) for k in ("bytes", "flops")}
    while True:
        n_kv = rng.choice([1, 2, 4, 8])
        cache = dict(n_kv=n_kv, hd=rng.choice([64, 128, 128, 256]),
                     page=rng.choice([16, 32, 64, 64, 128, 256]))
        heads = dict(n_q=n_kv * rng.choice([1, 2, 4, 7, 12]), **cache)
        dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
        batch = _log(rng, 1, 64)
        if op == "append":
            hi = rng.choice([1, _log(rng, 1, 2000)])
            case = _append("", dtype, batch, rng.choice([0, _log(rng, 1, 2000)]), _log(rng, 1, hi), hi,
                           rot=rng.choice([1, 1, 2]) * cache["hd"] // 2, norm=rng.random() < 0.5, **heads)
        elif op == "read":
            case = _read("", dtype, _log(rng, 1, 60000), **cache)
        elif op == "decode":
            tokens = rng.choice([1, 1, 1, rng.randint(2, 9)])
            hi = _log(rng, tokens, 32000)
            case = _decode("", dtype, batch, tokens, rng.choice([0, _log(rng, 1, 32000)]),
                           _log(rng, tokens, hi), hi, **heads)
        else:
            case = _verify("", dtype, batch, rng.randint(0, 9), _log(rng, 1000, 260000),
                           rng.choice([0.0, rng.uniform(0.1, 2)]), rng.random() < 0.7)
        del case["name"]
        w = work(case)
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"] and _plain_bytes(case) < 2e10:
            return case


def _plain_bytes(case):
    """What the plain forms of the attention and its padded tables take."""
    if case["op"] != "decode":
        return 0
    keys = case["hi"] + 512
    return 4.0 * (case["batch"] * case["tokens"] * case["n_q"] * (keys + case["prefix"])
                  + 4 * (case["batch"] * keys + case["prefix"]) * case["n_kv"] * case["hd"])


def _runs(case):
    """The batch's lengths: of the case alone, so that its work is."""
    rng = random.Random("%(batch)d %(lo)d %(hi)d" % case)
    runs = [case["hi"], case["lo"]] + [rng.randint(case["lo"], case["hi"])
                                      for _ in range(case["batch"])]
    return runs[:case["batch"]]


def work(case):
    e = _SIZE[case["dtype"]]
    if case["op"] == "verify":
        # the row of p behind the drafts that are kept, and the draft's own there
        rows = 2 if case["given"] and case["drafts"] else 1
        n = case["batch"] * case["vocab"]
        return {"bytes": n * rows * e + 64 * case["batch"], "flops": n * (rows + 2)}
    n_kv, hd = case["n_kv"], case["hd"]
    if case["op"] == "read":
        n = 2 * case["rows"] * n_kv * hd
        return {"bytes": n * (_STORED + e) + 8 * case["rows"], "flops": 2 * n}
    runs, n_q = _runs(case), case["n_q"]
    if case["op"] == "append":
        n = sum(runs)
        # queries in and out, keys and values in, into the cache and read back
        data = n * (2 * n_q * e + 2 * n_kv * (2 * e + _STORED)) * hd
        return {"bytes": data + max(runs) * case["rot"] * 4 + 16 * n,
                "flops": n * (n_q + 4 * n_kv) * hd * (7 if case["norm"] else 3)}
    keys, t = case["prefix"] + sum(runs), case["tokens"]
    pairs = t * (case["batch"] * case["prefix"] + sum(runs)) - case["batch"] * t * (t - 1) // 2
    return {"bytes": 2 * keys * n_kv * hd * _STORED + 2 * case["batch"] * t * n_q * hd * e,
            "flops": 4 * hd * n_q * pairs}


# ---- inputs -----------------------------------------------------------------

def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _pages_of(pool, count, width):
    """The next `count` pages of the pool, as a table row of `width` entries."""
    return [pool.pop() for _ in range(count)] + [-1] * (width - count)


def _cache(n_pages, n_kv, page, hd):
    """An empty pool: codes and scales of keys and values side by side."""
    codes = torch.zeros(n_pages, 2, n_kv, page, hd // 2, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(n_pages, 2, n_kv, page, hd // GROUP, 2, dtype=torch.bfloat16, device="cuda")
    return dict(k_codes=codes[:, 0], k_scales=scales[:, 0], v_codes=codes[:, 1], v_scales=scales[:, 1])


def _fill(cache, randn):
    """Random keys and values in every row, 16 pages at a time."""
    for name in ("k", "v"):
        codes, scales = cache[name + "_codes"], cache[name + "_scales"]
        for i in range(0, codes.shape[0], 16):
            x = randn(*codes[i:i + 16].shape[:3], 2 * codes.shape[3])
            codes[i:i + 16], scales[i:i + 16] = _quantised(x)


def prepare(case, seed):
    if own:
        _operators()                                # a program loads the library once
    rng = random.Random(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _TYPES[case["dtype"]]

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)

    if case["op"] == "verify":
        return _prepare_verify(case, g, randn, dt)
    page, n_kv, hd = case["page"], case["n_kv"], case["hd"]
    if case["op"] == "read":
        n = case["rows"]
        count = -(-n // page)
        pool = list(range(count + 3))
        rng.shuffle(pool)
        cache = _cache(len(pool), n_kv, page, hd)
        _fill(cache, randn)
        slots = [pool[i // page] * page + i % page for i in range(n)]
        return dict(op="read", slots=_ints(slots, torch.int64), dtype=dt, **cache)
    runs = _runs(case)
    past, prefix = case.get("past", 0), case.get("prefix", 0)
    lens = [past + t for t in runs]
    count = [-(-n // page) for n in lens]
    p_count = -(-prefix // page)
    n_pages = sum(count) + p_count + 3
    pool = list(range(n_pages))
    rng.shuffle(pool)
    width = max(count) + max(1, 256 // page)        # room for 256 more tokens
    prefix_table = _pages_of(pool, p_count, p_count)
    tables = [_pages_of(pool, n, width) for n in count]
    cache = _cache(n_pages, n_kv, page, hd)
    if case["op"] == "append":
        # one row-stacked q/k/v product, cut into its three parts
        n, n_q, rot = sum(runs), case["n_q"], case["rot"]
        y = randn(n, (n_q + 2 * n_kv) * hd, dtype=dt)
        q, k, v = (t.unflatten(1, (-1, hd)) for t in y.split([n_q * hd, n_kv * hd, n_kv * hd], 1))
        angles = (torch.arange(past + max(runs), dtype=torch.float64, device="cuda")[:, None]
                  * THETA ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot))
        angles = torch.cat([angles, angles], 1)
        positions = [past + p for t in runs for p in range(t)]
        slots = [row[p // page] * page + p % page for row, t in zip(tables, runs)
                 for p in range(past, past + t)]
        weights = [1 + 0.1 * randn(hd) for _ in range(2)]
        return dict(op="append", q=q, k=k, v=v, cos=angles.cos().float(), sin=angles.sin().float(),
                    positions=_ints(positions, torch.int64), slots=_ints(slots, torch.int64),
                    norm=case["norm"], q_weight=weights[0], k_weight=weights[1], dtype=dt, **cache)
    _fill(cache, randn)
    q = 1.5 * randn(case["batch"] * case["tokens"], case["n_q"], hd)
    return dict(op="decode", q=q.to(dt), prefix_table=_ints(prefix_table), prefix=prefix,
                tables=_ints(tables), lengths=_ints(lens), scale=hd ** -0.5, **cache)


def _prepare_verify(case, g, randn, dt):
    """Probabilities of a target and of a draft that is near it, and tokens drawn
    from the draft's."""
    B, K, V = case["batch"], case["drafts"], case["vocab"]
    logits = 2.5 * randn(B, K + 1, V)
    near = logits[:, :K] + case["spread"] * randn(B, K, V)
    drafted = torch.softmax(near, -1).to(dt)
    probs = torch.softmax(logits, -1).to(dt)
    del logits, near
    if K:
        drafts = torch.multinomial(drafted.flatten(0, 1).float(), 1, generator=g).view(B, K)
    else:
        drafts = torch.empty(B, 0, dtype=torch.int64, device="cuda")
    uniforms = torch.rand(B, K + 1, generator=g, device="cuda")
    return dict(op="verify", probs=probs, drafts=drafts,
                draft_probs=drafted if case["given"] and K else None, uniforms=uniforms)


# ---- the framework's operators ------------------------------------------------

def _operators():
    pkg = os.path.abspath("codebook-quantization_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import cbq_ops
    return cbq_ops.load()


def run(s):
    if not own:
        return {"append": _plain_append, "read": _plain_read, "decode": _plain_decode,
                "verify": _plain_verify}[s["op"]](s)
    ops = torch.ops.cbq
    if s["op"] == "verify":
        return ops.verify_drafts(s["probs"], s["drafts"], s["draft_probs"], None, s["uniforms"])
    cache = s["k_codes"], s["k_scales"], s["v_codes"], s["v_scales"]
    if s["op"] == "read":
        return ops.paged_read_q4(*cache, s["slots"], s["dtype"])
    if s["op"] == "append":
        q = ops.paged_append_q4(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["positions"],
                                s["slots"], *cache, s["norm"], s["q_weight"] if s["norm"] else None,
                                s["k_weight"] if s["norm"] else None, EPS)
        return q, *ops.paged_read_q4(*cache, s["slots"], s["dtype"])
    return ops.prefix_attention_decode_q4(s["q"], *cache, s["prefix_table"], s["prefix"],
                                          s["tables"], s["lengths"], s["scale"])


# ---- plain forms ----------------------------------------------------------------

def _quantised(x):
    """[..., hd] -> codes [..., hd / 2] and (scale, mid) [..., hd / 64, 2]: in 64
    bits, since a code next to a border has to come out the same everywhere."""
    x = x.double().unflatten(-1, (-1, GROUP))
    top, low = x.amax(-1), x.amin(-1)
    mid = ((top + low) / 2).float().bfloat16()
    m = mid.double()
    scale = (torch.maximum(top - m, m - low) / 7.5).float().bfloat16()
    s = scale.double()[..., None]
    c = torch.where(s > 0, torch.floor((x - m[..., None]) / s) + 8, 8.0).clamp(0, 15).to(torch.uint8)
    c = c.unflatten(-1, (-1, 4)).transpose(-3, -2).flatten(-3)      # four of each group in turn
    return c[..., 0::2] | c[..., 1::2] << 4, torch.stack([scale, mid], -1)


def _values(codes, scales):
    """[..., hd / 2] and [..., hd / 64, 2] -> [..., hd] in 32 bits."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    c = c.unflatten(-1, (GROUP // 4, -1, 4)).transpose(-3, -2).flatten(-2).float()
    return (scales[..., 1:].float() + scales[..., :1].float() * (c - 7.5)).flatten(-2)


def _plain_rotate(x, weight, s, dtype):
    x = x.to(dtype)
    if s["norm"]:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.to(dtype)
    half = s["cos"].shape[1] // 2
    c, n = (t[s["positions"], None, :half].to(dtype) for t in (s["cos"], s["sin"]))
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    return torch.cat([a * c - b * n, b * c + a * n, rest], -1)


def _plain_append(s):
    q = _plain_rotate(s["q"], s["q_weight"], s, torch.float32).to(s["dtype"])
    page = s["k_codes"].shape[2]
    at, row = s["slots"] // page, s["slots"] % page
    k = _plain_rotate(s["k"], s["k_weight"], s, torch.float64)
    s["k_codes"][at, :, row], s["k_scales"][at, :, row] = _quantised(k)
    s["v_codes"][at, :, row], s["v_scales"][at, :, row] = _quantised(s["v"])
    return q, *_plain_read(s)


def _plain_read(s):
    page = s["k_codes"].shape[2]
    at, row = s["slots"] // page, s["slots"] % page
    return tuple(_values(s[n + "_codes"][at, :, row], s[n + "_scales"][at, :, row]).to(s["dtype"])
                 for n in ("k", "v"))


def _dense(s, name, table):
    """[..., W] page ids -> [..., n_kv, W * page, hd] in 32 bits."""
    at = table.clamp(min=0).long()
    x = _values(s[name + "_codes"][at], s[name + "_scales"][at])
    return x.transpose(-4, -3).flatten(-3, -2)


def _softmax(scores):
    """exp(scores - max) and its sums; a row that sees nothing sums to 0."""
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    return p, p.sum(-1, keepdim=True)


def _plain_decode(s):
    N, n_q, hd = s["q"].shape
    n_kv, P, B = s["k_codes"].shape[1], s["prefix"], s["lengths"].shape[0]
    T, rep = N // B, n_q // n_kv
    q = s["q"].float().view(B, T, n_kv, rep, hd).permute(0, 2, 1, 3, 4)     # [B, n_kv, T, rep, hd]
    qp = q.transpose(0, 1).reshape(n_kv, B * T * rep, hd)       # the prefix: one product for all
    kp, vp = (_dense(s, t, s["prefix_table"])[:, :P] for t in ("k", "v"))
    sp = torch.matmul(qp, kp.transpose(1, 2).contiguous()).view(n_kv, B, T * rep, P).transpose(0, 1)
    ko = _dense(s, "k", s["tables"])
    so = torch.matmul(q.reshape(B, n_kv, T * rep, hd), ko.transpose(2, 3).contiguous())
    del ko
    last = s["lengths"][:, None] - T + torch.arange(T, device="cuda")       # [B, T]
    hidden = torch.arange(so.shape[-1], device="cuda") > last[:, :, None]
    hidden = hidden[:, None, :, None, :].expand(B, 1, T, rep, -1).reshape(B, 1, T * rep, -1)
    so = so.masked_fill(hidden, float("-inf"))
    p, total = _softmax(torch.cat([sp, so], -1) * s["scale"])
    pp = p[..., :P].transpose(0, 1).reshape(n_kv, B * T * rep, P)
    out = torch.matmul(pp, vp).view(n_kv, B, T * rep, hd).transpose(0, 1)
    out = out + torch.matmul(p[..., P:], _dense(s, "v", s["tables"]))
    out = out / torch.where(total == 0, 1.0, total)
    out = out.view(B, n_kv, T, rep, hd).transpose(1, 2).reshape(N, n_q, hd)
    return out.to(s["q"].dtype)


def _plain_verify(s):
    """Products, differences and cumulative sums in 64 bits: a random number next
    to a border has to fall on the same side everywhere."""
    p, q, drafts, u = s["probs"], s["draft_probs"], s["drafts"], s["uniforms"].double()
    B, K = drafts.shape
    V = p.shape[2]
    b = torch.arange(B, device="cuda")
    at = drafts.clamp(0, V - 1)[..., None]
    inside = (drafts >= 0) & (drafts < V)
    pd = torch.where(inside, p[:, :K].gather(2, at)[..., 0].double(), 0.0)
    qd = q.gather(2, at)[..., 0].double() if q is not None else torch.ones_like(pd)
    kept = (u[:, :K] * qd < pd).long().cumprod(1).sum(1)        # drafts before the first refused
    row = p[b, kept].double()
    if K:
        refused = (kept < K)[:, None]
        i = kept.clamp(max=K - 1)
        if q is not None:
            less = q[b, i].double()
        else:
            less = (torch.arange(V, device="cuda") == drafts[b, i][:, None]) * row
        rest = torch.where(refused, row - less, row)
    else:
        rest = row
    rest, row = (torch.where(x > 0, x, 0.0) for x in (rest, row))
    rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, row)
    sums = rest.cumsum(1)
    token = (sums <= u[:, K:] * sums[:, -1:]).sum(1)
    last = (torch.arange(1, V + 1, device="cuda") * (rest > 0)).amax(1) - 1
    token = torch.minimum(token, last)
    n = torch.arange(K + 1, device="cuda")
    tokens = torch.cat([drafts, drafts.new_zeros(B, 1)], 1)
    tokens = torch.where(n == kept[:, None], token[:, None], tokens)
    return torch.where(n <= kept[:, None], tokens, -1), (kept + 1).int()


# ---- the definitions in 64 bits -------------------------------------------------

def _step(x):
    """Nearest bf16 number of 64-bit values, through fp32."""
    return x.to(torch.float32).to(torch.bfloat16).to(torch.float64)


def _exact_stored(x):
    """What a row stands for once it is stored, group by group: its range cut into
    15 half-open steps about the middle, each value the centre of its step."""
    out = torch.empty_like(x)
    for i in range(0, x.shape[-1], GROUP):
        y = x[..., i:i + GROUP]
        low, high = torch.aminmax(y, dim=-1, keepdim=True)
        middle = _step(low + (high - low) / 2)
        step = _step(torch.max(high - middle, middle - low) / 7.5)
        n = torch.div(y - middle, torch.where(step > 0, step, 1.0), rounding_mode="floor")
        out[..., i:i + GROUP] = middle + step * (n.clamp(-8, 7) + 0.5)
    return out


def _exact_append(s):
    """Each head as complex numbers turned by its position's angle."""
    def turned(x, weight):
        x = x.double()
        if s["norm"]:
            x = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * weight.double()
        rot = s["cos"].shape[1]
        z = torch.complex(x[..., :rot // 2], x[..., rot // 2:rot])
        turn = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"], :rot // 2]
        z = z * turn[:, None]
        return torch.cat([z.real, z.imag, x[..., rot:]], -1)

    return (turned(s["q"], s["q_weight"]), _exact_stored(turned(s["k"], s["k_weight"])),
            _exact_stored(s["v"].double()))


def _exact_rows(codes, scales, places):
    """Rows (page, row) of one head, from its bytes [n_pages, page, hd / 2]."""
    page = codes.shape[1]
    byte = codes.reshape(-1, codes.shape[2])[places].long()
    pair = scales.reshape(codes.shape[0] * page, -1, 2)[places].double()
    hd = 2 * byte.shape[1]
    d = torch.arange(hd, device="cuda")
    g, e = d // GROUP, d % GROUP
    half = byte[:, e // 4 * (hd // 32) + 2 * g + e % 4 // 2]
    code = torch.where(e % 2 == 0, half % 16, torch.div(half, 16, rounding_mode="floor")).double()
    each = pair.repeat_interleave(GROUP, 1)
    return (2 * code - 15) / 2 * each[..., 0] + each[..., 1]


def _exact_read(s):
    return tuple(torch.stack([_exact_rows(s[n + "_codes"][:, h], s[n + "_scales"][:, h], s["slots"])
                              for h in range(s["k_codes"].shape[1])], 1) for n in ("k", "v"))


def _exact_decode(s):
    """Sequence by sequence and head by head."""
    N, n_q, hd = s["q"].shape
    n_kv, page = s["k_codes"].shape[1], s["k_codes"].shape[2]
    rep = n_q // n_kv
    out = torch.zeros(N, n_q, hd, dtype=torch.float64, device="cuda")
    lens, rows = s["lengths"].tolist(), s["tables"]
    T = N // len(lens)

    def places(table, n):
        j = torch.arange(n, device="cuda")
        return table.long()[j // page] * page + j % page

    shared = places(s["prefix_table"], s["prefix"])
    for b, length in enumerate(lens):
        at = torch.cat([shared, places(rows[b], length)])
        seen = len(at) - T + 1 + torch.arange(T, device="cuda")
        hidden = torch.arange(len(at), device="cuda")[None] >= seen[:, None]
        mine = slice(b * T, (b + 1) * T)
        for h in range(n_kv):
            k, v = (_exact_rows(s[n + "_codes"][:, h], s[n + "_scales"][:, h], at) for n in ("k", "v"))
            for i in range(h * rep, (h + 1) * rep):
                w = (s["q"][mine, i].double() @ k.t() * s["scale"]).masked_fill(hidden, -math.inf)
                w = (w - w.max(1, keepdim=True).values).exp()
                out[mine, i] = (w / w.sum(1, keepdim=True)) @ v
    return out


def _exact_verify(s):
    """Draft by draft, as the rule is told; the last token by a search in the sums."""
    B, K = s["drafts"].shape
    V = s["probs"].shape[2]
    tokens, counts = [], []
    for b, line in enumerate(s["drafts"].tolist()):
        u = s["uniforms"][b].double().tolist()
        said = []
        for i, d in enumerate(line):
            p = float(s["probs"][b, i, d])
            q = float(s["draft_probs"][b, i, d]) if s["draft_probs"] is not None else 1.0
            if not u[i] * q < p:
                break
            said.append(d)
        i = len(said)
        p = s["probs"][b, i].double()
        left = p.clone()
        if i < K and s["draft_probs"] is not None:
            left -= s["draft_probs"][b, i].double()
        elif i < K:
            left[line[i]] = 0
        left = left.clamp(min=0)
        if not left.any():
            left = p
        sums = left.cumsum(0)
        at = int(torch.searchsorted(sums, (u[K] * sums[-1]).reshape(1), right=True))
        said.append(min(at, int(left.nonzero().max())))
        counts.append(len(said))
        tokens.append(said + [-1] * (K + 1 - len(said)))
    return _ints(tokens, torch.int64), _ints(counts)


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "read": _exact_read, "decode": _exact_decode,
            "verify": _exact_verify}[s["op"]](s)
