"""Serving a batch over a paged key/value cache, as measurable cases.

Three operators of torch.ops.cbq (cbq_ops.load()), each with its plain form in
elementary torch operations in 32 bits:

- "append": paged_append, the head norm and rotation of new tokens' queries
  and keys, and the keys and values into their pages;
- "decode": prefix_attention_decode, one query token for each sequence of a
  batch that shares a prefix (computed once for all of them);
- "prompt": prefix_attention_prompt, ragged runs of new tokens of such a
  batch, causal over their own keys.

Pages are [n_pages, n_kv, page, hd], scattered over a pool; a table row names
a sequence's pages in order and has room to grow (-1 where no page is taken
yet).  Head layouts are those of the two decoder configurations of
codebook-quantization_amd/synthetic.py (32 and 16 query heads on 8 kv heads of
128) and generic ones of the other head sizes.
"""
import math
import os
import random
import sys

import torch

own = False                  # True: run() calls the framework's operators

EPS = 1.0e-6
THETA = 1.0e6
_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def _append(name, dtype, cache, batch, past, lo, hi, n_q, n_kv, hd, page, rot=None, norm=True):
    """batch runs of lo..hi new tokens each, behind `past` cached ones."""
    return dict(name=name, op="append", dtype=dtype, cache=cache, batch=batch, past=past, lo=lo,
                hi=hi, n_q=n_q, n_kv=n_kv, hd=hd, page=page, rot=rot or hd, norm=norm)


def _decode(name, dtype, batch, prefix, lo, hi, n_q, n_kv, hd, page):
    """batch sequences of lo..hi own keys each behind `prefix` shared ones."""
    return dict(name=name, op="decode", dtype=dtype, batch=batch, prefix=prefix, lo=lo, hi=hi,
                n_q=n_q, n_kv=n_kv, hd=hd, page=page)


def _prompt(name, dtype, batch, prefix, past, lo, hi, n_q, n_kv, hd, page):
    """batch runs of lo..hi new tokens, behind `past` own keys and `prefix` shared ones."""
    return dict(name=name, op="prompt", dtype=dtype, batch=batch, prefix=prefix, past=past, lo=lo,
                hi=hi, n_q=n_q, n_kv=n_kv, hd=hd, page=page)


def listed():
    return [
        # one token of one sequence of the fp32 decoder, 8B head layout: latency
        _append("append-1-f32", "f32", "f32", 1, 383, 1, 1, 32, 8, 128, 16),
        # a decode step of a large batch, bf16 model of the 8B head layout
        _append("append-64x1-bf16", "bf16", "bf16", 64, 200, 1, 1, 32, 8, 128, 64),
        # the fp32 decoder with a bf16 cache, 1.7B head layout, half of each
        # head rotated: a few short prompts
        _append("append-prompts-f32-to-bf16", "f32", "bf16", 7, 0, 11, 250, 16, 8, 128, 32,
                rot=64, norm=False),
        # a scheduler's pass over many prompts at once
        _append("append-prompts-bf16", "bf16", "bf16", 24, 0, 40, 1000, 32, 8, 128, 64),
        # one sequence of the fp32 decoder after its 128-token prompt and 256
        # tokens, no prefix: latency
        _decode("decode-1x384-f32", "f32", 1, 0, 384, 384, 32, 8, 128, 16),
        # a batch behind a system prompt, 1.7B head layout
        _decode("decode-16-bf16-prefix1000", "bf16", 16, 1000, 100, 400, 16, 8, 128, 32),
        # many questions about one long document, 8B head layout: the largest
        _decode("decode-64-bf16-prefix30011", "bf16", 64, 30011, 200, 1500, 32, 8, 128, 64),
        # heads of 64 in groups of twelve, very uneven lengths, fp16
        _decode("decode-33-f16-prefix5000", "f16", 33, 5000, 1, 2900, 24, 2, 64, 128),
        # the fp32 decoder's prompt, 1.7B head layout, no prefix
        _prompt("prompt-200-f32", "f32", 1, 0, 0, 200, 200, 16, 8, 128, 16),
        # ragged questions behind a shared system prompt, 8B head layout
        _prompt("prompts-16-bf16-prefix2048", "bf16", 16, 2048, 0, 20, 600, 32, 8, 128, 64),
        # a chunk of a long conversation with heads of 256: few rows, many keys
        _prompt("chunks-2-f16-past20000", "f16", 2, 0, 20000, 33, 64, 8, 2, 256, 256),
        # one long document read in, 8B head layout: the most arithmetic
        _prompt("prompt-8192-bf16", "bf16", 1, 0, 0, 8192, 8192, 32, 8, 128, 64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges, no larger than its operator's largest."""
    op = rng.choice(["append", "decode", "prompt"])
    most = max((work(c) for c in listed() if c["op"] == op), key=lambda w: w["bytes"] + w["flops"])
    while True:
        hd = rng.choice([64, 128, 128, 256])
        n_kv = rng.choice([1, 2, 4, 8])
        heads = dict(n_q=n_kv * rng.choice([1, 2, 4, 7, 12]), n_kv=n_kv, hd=hd,
                     page=rng.choice([16, 32, 64, 128, 256]))
        dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
        batch = _log(rng, 1, 64)
        prefix = rng.choice([0, _log(rng, 1, 32000)])
        if op == "append":
            hi = rng.choice([1, _log(rng, 1, 2000)])
            cache = rng.choice(["f32", "bf16", "f16"]) if dtype == "f32" else dtype
            case = _append("", dtype, cache, batch, rng.choice([0, _log(rng, 1, 2000)]),
                           _log(rng, 1, hi), hi, rot=rng.choice([hd, hd, hd // 2]),
                           norm=rng.random() < 0.5, **heads)
        elif op == "decode":
            hi = _log(rng, 1, 8000)
            case = _decode("", dtype, batch, prefix, _log(rng, 1, hi), hi, **heads)
        else:
            hi = _log(rng, 2, 6000)
            case = _prompt("", dtype, max(1, batch // 4), prefix,
                           rng.choice([0, _log(rng, 1, 20000)]), _log(rng, 1, hi), hi, **heads)
        del case["name"]
        w = work(case)
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"] and _plain_bytes(case) < 3e10:
            return case


def _plain_bytes(case):
    """What the plain form's padded scores take."""
    if case["op"] == "append":
        return 0
    keys = case["prefix"] + case.get("past", 0) + case["hi"] + 256
    rows = case["batch"] * (case["hi"] if case["op"] == "prompt" else 1)
    return 4.0 * rows * case["n_q"] * keys


def _runs(case):
    """The batch's lengths: of the case alone, so that its work is."""
    rng = random.Random("%(batch)d %(lo)d %(hi)d" % case)
    runs = [case["hi"], case["lo"]] + [rng.randint(case["lo"], case["hi"])
                                      for _ in range(case["batch"])]
    return runs[:case["batch"]]


def work(case):
    runs, e = _runs(case), _SIZE[case["dtype"]]
    n_q, n_kv, hd = case["n_q"], case["n_kv"], case["hd"]
    if case["op"] == "append":
        n, c = sum(runs), _SIZE[case["cache"]]
        data = n * (n_q + 2 * n_kv) * hd * (e + c)
        return {"bytes": data + max(runs) * case["rot"] * 4 + 16 * n,
                "flops": n * (n_q + n_kv) * hd * (7 if case["norm"] else 3)}
    if case["op"] == "decode":
        keys, pairs, n = case["prefix"] + sum(runs), case["batch"] * case["prefix"] + sum(runs), \
            case["batch"]
    else:
        keys, n = case["prefix"] + sum(case["past"] + t for t in runs), sum(runs)
        pairs = sum(t * (case["prefix"] + case["past"]) + t * (t + 1) // 2 for t in runs)
    return {"bytes": (2 * keys * n_kv + 2 * n * n_q) * hd * e, "flops": 4 * hd * n_q * pairs}


# ---- inputs -----------------------------------------------------------------

def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _pages_of(pool, count, width):
    """The next `count` pages of the pool, as a table row of `width` entries."""
    return [pool.pop() for _ in range(count)] + [-1] * (width - count)


def prepare(case, seed):
    if own:
        _operators()                                # a program loads the library once
    rng = random.Random(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    runs, page, n_kv, hd = _runs(case), case["page"], case["n_kv"], case["hd"]
    dt = _TYPES[case["dtype"]]
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
    shape = (n_pages, 2, n_kv, page, hd)

    def randn(*shape, dtype=dt):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)

    if case["op"] == "append":
        # one row-stacked q/k/v product, cut into its three parts
        n, n_q, rot = sum(runs), case["n_q"], case["rot"]
        y = randn(n, (n_q + 2 * n_kv) * hd)
        q, k, v = (t.unflatten(1, (-1, hd)) for t in y.split([n_q * hd, n_kv * hd, n_kv * hd], 1))
        angles = (torch.arange(past + max(runs), dtype=torch.float64, device="cuda")[:, None]
                  * THETA ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot))
        angles = torch.cat([angles, angles], 1)
        cache = randn(*shape, dtype=_TYPES[case["cache"]])
        positions = [past + p for t in runs for p in range(t)]
        slots = [row[p // page] * page + p % page for row, t in zip(tables, runs)
                 for p in range(past, past + t)]
        weights = [1 + 0.1 * randn(hd, dtype=torch.float32) for _ in range(2)]
        return dict(op="append", q=q, k=k, v=v, cos=angles.cos().float(),
                    sin=angles.sin().float(), positions=_ints(positions, torch.int64),
                    slots=_ints(slots, torch.int64), k_pages=cache[:, 0], v_pages=cache[:, 1],
                    norm=case["norm"], q_weight=weights[0], k_weight=weights[1])
    n = sum(runs) if case["op"] == "prompt" else case["batch"]
    cache = randn(*shape)
    starts = [sum(runs[:i]) for i in range(len(runs) + 1)]
    return dict(op=case["op"], q=1.5 * randn(n, case["n_q"], hd), k_pages=cache[:, 0],
                v_pages=cache[:, 1], prefix_table=_ints(prefix_table), prefix=prefix,
                tables=_ints(tables), lengths=_ints(lens), q_start=_ints(starts),
                longest=max(runs), scale=hd ** -0.5)


# ---- the framework's operators ------------------------------------------------

def _operators():
    pkg = os.path.abspath("codebook-quantization_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import cbq_ops
    return cbq_ops.load()


def run(s):
    if not own:
        return {"append": _plain_append, "decode": _plain_decode,
                "prompt": _plain_prompt}[s["op"]](s)
    ops = torch.ops.cbq
    if s["op"] == "append":
        q = ops.paged_append(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["positions"],
                             s["slots"], s["k_pages"], s["v_pages"], s["norm"],
                             s["q_weight"] if s["norm"] else None,
                             s["k_weight"] if s["norm"] else None, EPS)
        return q, s["k_pages"], s["v_pages"]
    if s["op"] == "decode":
        return ops.prefix_attention_decode(s["q"], s["k_pages"], s["v_pages"], s["prefix_table"],
                                           s["prefix"], s["tables"], s["lengths"], s["scale"])
    return ops.prefix_attention_prompt(s["q"], s["q_start"], s["k_pages"], s["v_pages"],
                                       s["prefix_table"], s["prefix"], s["tables"], s["lengths"],
                                       s["scale"])


# ---- plain forms ----------------------------------------------------------------

def _plain_rotate(x, weight, s):
    x = x.float()
    if s["norm"]:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight
    half = s["cos"].shape[1] // 2
    c, n = (t[s["positions"], None, :half] for t in (s["cos"], s["sin"]))
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    return torch.cat([a * c - b * n, b * c + a * n, rest], -1).to(s["k_pages"].dtype)


def _plain_append(s):
    q = _plain_rotate(s["q"], s["q_weight"], s)
    page = s["k_pages"].shape[2]
    at, row = s["slots"] // page, s["slots"] % page
    s["k_pages"][at, :, row] = _plain_rotate(s["k"], s["k_weight"], s)
    s["v_pages"][at, :, row] = s["v"].to(s["v_pages"].dtype)
    return q, s["k_pages"], s["v_pages"]


def _dense(pages, table):
    """[..., W] page ids -> [..., n_kv, W * page, hd] in 32 bits."""
    x = pages[table.clamp(min=0).long()].float().transpose(-4, -3)
    return x.flatten(-3, -2)


def _softmax(scores):
    """exp(scores - max) and its sums; a row that sees nothing sums to 0."""
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    return p, p.sum(-1, keepdim=True)


def _plain_decode(s):
    B, n_q, hd = s["q"].shape
    n_kv, P = s["k_pages"].shape[1], s["prefix"]
    rep = n_q // n_kv
    q = s["q"].float().view(B, n_kv, rep, hd)
    qp = q.transpose(0, 1).reshape(n_kv, B * rep, hd)           # the prefix: one product for all
    kp, vp = (_dense(t, s["prefix_table"])[:, :P] for t in (s["k_pages"], s["v_pages"]))
    sp = torch.matmul(qp, kp.transpose(1, 2).contiguous()).view(n_kv, B, rep, P).transpose(0, 1)
    ko, vo = (_dense(t, s["tables"]) for t in (s["k_pages"], s["v_pages"]))
    so = torch.matmul(q, ko.transpose(2, 3).contiguous())
    hidden = torch.arange(so.shape[-1], device="cuda") >= s["lengths"][:, None, None, None]
    so = so.masked_fill(hidden, float("-inf"))
    p, total = _softmax(torch.cat([sp, so], -1) * s["scale"])
    pp = p[..., :P].transpose(0, 1).reshape(n_kv, B * rep, P)
    out = torch.matmul(pp, vp).view(n_kv, B, rep, hd).transpose(0, 1)
    out = (out + torch.matmul(p[..., P:], vo)) / torch.where(total == 0, 1.0, total)
    return out.reshape(B, n_q, hd).to(s["q"].dtype)


def _plain_prompt(s):
    N, n_q, hd = s["q"].shape
    n_kv, P, T = s["k_pages"].shape[1], s["prefix"], s["longest"]
    start, count = s["q_start"][:-1].long(), s["q_start"].diff()
    B, rep = count.numel(), n_q // n_kv
    t = torch.arange(T, device="cuda")
    q = s["q"][(start[:, None] + t).clamp(max=N - 1)].float()       # [B, T, n_q, hd], padded
    q = q.view(B, T, n_kv, rep, hd).permute(0, 2, 1, 3, 4).reshape(B, n_kv, T * rep, hd)
    kp, vp = (_dense(x, s["prefix_table"])[:, :P] for x in (s["k_pages"], s["v_pages"]))
    ko, vo = (_dense(x, s["tables"]) for x in (s["k_pages"], s["v_pages"]))
    scores = torch.cat([torch.matmul(q, kp.transpose(1, 2).contiguous()),
                        torch.matmul(q, ko.transpose(2, 3).contiguous())], -1) * s["scale"]
    last = (s["lengths"] - count)[:, None] + t                      # [B, T]
    hidden = torch.arange(ko.shape[2], device="cuda") > last[:, :, None]
    hidden = hidden[:, None, :, None, :].expand(B, 1, T, rep, -1).reshape(B, 1, T * rep, -1)
    scores[..., P:].masked_fill_(hidden, float("-inf"))
    p, total = _softmax(scores)
    out = torch.matmul(p[..., :P], vp) + torch.matmul(p[..., P:], vo)
    out = out / torch.where(total == 0, 1.0, total)
    out = out.view(B, n_kv, T, rep, hd).transpose(1, 2).reshape(B, T, n_q, hd)
    n = torch.arange(N, device="cuda")
    b = torch.searchsorted(s["q_start"][1:].long(), n, right=True)
    return out[b, n - start[b]].to(s["q"].dtype)


# ---- the definitions in 64 bits -------------------------------------------------

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

    def stored(pages, rows):
        n_pages, n_kv, page, hd = pages.shape
        flat = pages.double().permute(0, 2, 1, 3).reshape(n_pages * page, n_kv, hd).clone()
        flat.index_copy_(0, s["slots"], rows)
        return flat.view(n_pages, page, n_kv, hd).permute(0, 2, 1, 3).contiguous()

    return (turned(s["q"], s["q_weight"]), stored(s["k_pages"], turned(s["k"], s["k_weight"])),
            stored(s["v_pages"], s["v"].double()))


def _exact_attention(s):
    """Sequence by sequence and head by head."""
    N, n_q, hd = s["q"].shape
    n_kv, page = s["k_pages"].shape[1], s["k_pages"].shape[2]
    rep = n_q // n_kv
    out = torch.zeros(N, n_q, hd, dtype=torch.float64, device="cuda")
    lens = s["lengths"].tolist()
    ends = s["q_start"].tolist() if s["op"] == "prompt" else list(range(N + 1))
    shared = s["prefix_table"].tolist()
    rows = s["tables"].tolist()
    for b, length in enumerate(lens):
        mine = rows[b][:-(-length // page)]
        tokens = range(ends[b], ends[b + 1])
        place = torch.cat([torch.arange(s["prefix"]), len(shared) * page + torch.arange(length)])
        seen = s["prefix"] + length - len(tokens) + torch.arange(len(tokens)) + 1
        hidden = (torch.arange(len(place))[None] >= seen[:, None]).cuda()
        for h in range(n_kv):
            k, v = (x[shared + mine, h].double().reshape(-1, hd)[place.cuda()]
                    for x in (s["k_pages"], s["v_pages"]))
            for i in range(h * rep, (h + 1) * rep):
                w = s["q"][tokens.start:tokens.stop, i].double() @ k.t() * s["scale"]
                w = w.masked_fill(hidden, -math.inf)
                w = (w - w.max(1, keepdim=True).values).exp()
                out[tokens.start:tokens.stop, i] = (w / w.sum(1, keepdim=True)) @ v
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_append(s) if case["op"] == "append" else _exact_attention(s)
