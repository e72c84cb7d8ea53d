"""The operators of serving a batch of sequences, as timed cases.

A server that runs many sequences keeps their keys and values in pages of 8-bit
codes, attends to them from prompt rows and from single new tokens, computes a
long prefix that its sequences share once for all, and draws the next tokens.
Each case is one pass through one of these operators:

    cache      quantise new rows' keys and values into their sequences' pages
               and read them back
    attention  the rows' attention over their own sequences' pages
    prefix     the same for a batch whose sequences begin with the same pages
    sample     the next tokens from logits, by temperature, top-k, top-p and
               min-p, from given random numbers

With `own` false a pass computes the operator in elementary torch operations,
with `own` true by the library (gemma_hip.GemmaHip).  Widths are those of the
configurations in model_bin.

The formulas.  A row of `hdim` values of a head is stored as codes and one fp32
scale.  int8: scale = amax (1/127), code = x (127/amax) rounded to nearest, halves
away from zero.  e4m3: scale = amax (1/448), code = x (448/amax) rounded to
nearest, ties to even.  Every operation is one fp32 rounding; a row of zeros has
scale 0.  A value is code * scale.

Row i of a sequence's n new rows sits at position p = len - n + i and sees the
keys max(0, p + 1 - slide) .. p (slide 0: from 0).  Its head h reads kv head
h / (heads / kv): s = q.k asc, capped as cap tanh(s / cap) if cap is not 0;
out = sum softmax(s) v.

A row of logits l with temperature T, k, p, min-p and u: w = exp((l - max l) / T),
in the order of falling l, ties by rising index.  Kept are the first k, of these the
fewest whose w sum to at least p times theirs, and of these those with w >= min-p.
The token is the first whose running sum exceeds u times the sum of the kept ones,
its probability w over that sum.  T = 0 takes the first.
"""

from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

I8, E4M3 = "i8", "e4m3"
TOP = {I8: 127.0, E4M3: 448.0}


def listed():
    return [
        # one decode step of eight gemma-3-1b sequences into a layer's cache: the smallest, all latency
        dict(name="cache_step_1b", op="cache", batch=8, rows=1, ragged=False, len=1001, kv=1,
             hdim=256, page=16, type=I8),
        # four prompts of different lengths into a layer of gemma-3-4b, bandwidth
        dict(name="cache_prompts_4b", op="cache", batch=4, rows=4096, ragged=True, len=4096, kv=4,
             hdim=256, page=64, type=E4M3),
        # one new token of one gemma-3-1b sequence in a global layer, latency
        dict(name="step_1b_1001", op="attention", batch=1, rows=1, ragged=False, len=1001, heads=4,
             kv=1, hdim=256, page=16, slide=0, cap=0.0, type=I8),
        # a decode step of 32 gemma-3-4b sequences of different lengths
        dict(name="step_4b_32", op="attention", batch=32, rows=1, ragged=True, len=8192, heads=8,
             kv=4, hdim=256, page=64, slide=0, cap=0.0, type=I8),
        # two sequences at gemma-3's full context, the longest axis
        dict(name="step_1b_131072", op="attention", batch=2, rows=1, ragged=False, len=131072,
             heads=4, kv=1, hdim=256, page=256, slide=0, cap=0.0, type=E4M3),
        # two whole prompts through a sliding layer of gemma-3-4b
        dict(name="prompt_4b_sliding", op="attention", batch=2, rows=2048, ragged=False, len=2048,
             heads=8, kv=4, hdim=256, page=64, slide=1024, cap=0.0, type=I8),
        # an odd chunk of a prompt behind a filled cache, capped scores
        dict(name="prompt_1b_613", op="attention", batch=1, rows=613, ragged=False, len=2000,
             heads=4, kv=1, hdim=256, page=32, slide=0, cap=50.0, type=E4M3),
        # 64 questions behind one long document, gemma-3-1b
        dict(name="prefix_1b_64", op="prefix", batch=64, rows=1, ragged=True, shared=16384, len=513,
             heads=4, kv=1, hdim=256, page=64, slide=0, cap=0.0, type=I8),
        # 24 sequences behind a system prompt and its documents, gemma-3-4b
        dict(name="prefix_4b_24", op="prefix", batch=24, rows=1, ragged=True, shared=32768, len=300,
             heads=8, kv=4, hdim=256, page=64, slide=0, cap=0.0, type=E4M3),
        # one token of a chat: the usual filters over the whole vocabulary
        dict(name="sample_1", op="sample", rows=1, vocab=262144, spread=3.0, temperature=0.8,
             top_k=64, top_p=0.95, min_p=0.0),
        # a flat distribution cut by top-p alone: the kept set is tens of thousands
        dict(name="sample_7_flat", op="sample", rows=7, vocab=262144, spread=1.5, temperature=1.3,
             top_k=0, top_p=0.9, min_p=0.0),
        # a served batch, every row with settings of its own
        dict(name="sample_64_mixed", op="sample", rows=64, vocab=262144, spread=2.5, temperature=1.0,
             top_k=-1, top_p=0.9, min_p=0.05),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["cache", "cache", "attention", "attention", "attention", "attention",
                     "prefix", "prefix", "sample", "sample"])
    if op == "sample":
        rows = _log(rng, 1, 64)
        return dict(op=op, rows=rows, vocab=_log(rng, 1000, 262144),
                    spread=round(rng.uniform(0.5, 5.0), 2),
                    temperature=rng.choice([0.0, 0.5, 0.7, 1.0, 1.5]),
                    top_k=rng.choice([-1, 0, 1, 40, _log(rng, 2, 5000)]),
                    top_p=rng.choice([0.5, 0.9, 0.95, 1.0]), min_p=rng.choice([0.0, 0.0, 0.02, 0.1]))
    heads, kv, hdim = rng.choice([(4, 1, 256), (8, 4, 256), (4, 2, 128)])
    c = dict(op=op, kv=kv, hdim=hdim, page=rng.choice([16, 32, 64, 256]),
             type=rng.choice([I8, E4M3]))
    if op == "cache":
        rows = _log(rng, 1, 4096)
        batch = _log(rng, 1, max(1, min(64, 16384 // rows)))
        return dict(c, batch=batch, rows=rows, ragged=batch > 1 and rows > 1,
                    len=rows + rng.randint(0, 3000))
    c.update(heads=heads, slide=rng.choice([0, 0, 512, 1024]), cap=rng.choice([0.0, 0.0, 50.0]))
    if op == "prefix":
        c["batch"] = _log(rng, 2, 64)
        return dict(c, rows=rng.choice([1, 1, 1, rng.randint(2, 8)]), ragged=True,
                    shared=_log(rng, 256, 16384), len=_log(rng, 9, 600))
    if rng.random() < 0.5:  # single tokens
        c["batch"] = _log(rng, 1, 64)
        return dict(c, rows=1, ragged=rng.random() < 0.7,
                    len=_log(rng, 17, min(131072, 262144 // c["batch"])))
    rows = _log(rng, 2, 2048)
    return dict(c, batch=rng.randint(1, max(1, min(8, 4096 // rows))), rows=rows, ragged=False,
                len=rows + rng.choice([0, 0, rng.randint(1, 2000)]))


# ---- a case's sequences --------------------------------------------------------


def _spread(n, batch):
    """`batch` sizes from about n / 4 to n, in no order."""
    return [max(1, int(n * (0.25 + 0.75 * ((b * 0.6180339887) % 1.0)))) for b in range(batch)]


def _sequences(case):
    """New rows and length of every sequence."""
    b, n, ln = case["batch"], case["rows"], case["len"]
    if case["op"] == "cache":
        rows = _spread(n, b) if case["ragged"] else [n] * b
        return rows, [r + ln - n for r in rows]
    lens = _spread(ln, b) if case["ragged"] else [ln] * b
    lens = [max(n, x) + case.get("shared", 0) for x in lens]
    return [n] * b, lens


def _seen(case):
    """(first, last) key of every row, sequence by sequence."""
    out = []
    for n, ln in zip(*_sequences(case)):
        out.append([(max(0, p + 1 - case["slide"]) if case["slide"] else 0, p)
                    for p in range(ln - n, ln)])
    return out


# ---- inputs --------------------------------------------------------------------

_gh = None


def _lib():
    """The binding and the library's handle: one per process, on the first GPU."""
    global _gh
    # the package's folder has a dot in its name, so its modules go by path
    pkg = os.path.join(os.getcwd(), "gemma.c_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import gemma_hip

    if _gh is None:
        torch.cuda.init()
        _gh = gemma_hip.GemmaHip(0)
    return gemma_hip, _gh


def _unit(t):
    return t / t.square().mean(-1, keepdim=True).sqrt()


def _codes(x, kind):
    """Codes (as the type that holds them) and scales of rows x [..., hdim]."""
    amax = x.abs().amax(-1)
    inv = torch.where(amax > 0, (TOP[kind] / amax.double()), 1.0).float()
    scale = amax * torch.tensor(1.0 / TOP[kind], dtype=torch.float32, device=x.device)
    y = x * inv[..., None]
    if kind == I8:
        return torch.trunc(y + torch.copysign(torch.full_like(y, 0.5), y)).to(torch.int8), scale
    return y.clamp(-TOP[kind], TOP[kind]).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        st = dict(case=dict(case), logits=randn(rows, vocab) * case["spread"],
                  u=torch.rand(rows, generator=g, device="cuda"))

        def setting(name, dtype, other):
            if case["top_k"] >= 0:  # one setting for all rows
                return torch.full((rows,), case[name], dtype=dtype, device="cuda")
            i = torch.arange(rows, device="cuda")
            return torch.tensor(other, device="cuda", dtype=dtype)[i % len(other)].contiguous()

        t, p, m = case["temperature"], case["top_p"], case["min_p"]
        st.update(t=setting("temperature", torch.float32, [t, 0.7, t, 0.0, 1.5]),
                  k=setting("top_k", torch.int32, [0, 40, 1000, 1, 64, 0, 20000]),
                  p=setting("top_p", torch.float32, [1.0, p, 0.5]),
                  m=setting("min_p", torch.float32, [0.0, m]),
                  tokens=torch.empty(rows, dtype=torch.int32, device="cuda"),
                  probs=torch.empty(rows, device="cuda"))
        if own:
            gemma_hip, gh = _lib()
            st.update(settings=gemma_hip.sampling(st["t"], st["k"], st["p"], st["m"]),
                      work=torch.empty(gh.sample_work(rows, vocab), dtype=torch.uint8,
                                       device="cuda"))
        return st

    kv, hd, page, kind, batch = (case[f] for f in ("kv", "hdim", "page", "type", "batch"))
    rows, lens = _sequences(case)
    shared = case.get("shared", 0) // page  # whole pages that all sequences begin with
    need = [-(-ln // page) for ln in lens]
    width = max(need)
    npages = shared + sum(n - shared for n in need)
    order = torch.randperm(npages, generator=torch.Generator().manual_seed(seed))
    table = torch.zeros((batch, width), dtype=torch.int32)
    at = shared
    for b in range(batch):
        table[b, :shared] = order[:shared].int()
        table[b, shared:need[b]] = order[at:at + need[b] - shared].int()
        at += need[b] - shared
    ends = np.concatenate([[0], np.cumsum(rows)])
    st = dict(case=dict(case), seqs=(rows, lens), table=table.cuda(),
              row0=torch.tensor(ends, dtype=torch.int32, device="cuda"),
              len=torch.tensor(lens, dtype=torch.int32, device="cuda"),
              pos=torch.tensor(np.concatenate([np.arange(ln - n, ln) for n, ln in zip(rows, lens)]),
                               device="cuda"),
              seq=torch.tensor(np.repeat(np.arange(batch), rows), device="cuda"))
    dtype = torch.int8 if kind == I8 else torch.float8_e4m3fn
    for name in ("k", "v"):
        codes = torch.zeros((npages, kv, page, hd), dtype=torch.int8, device="cuda").view(dtype)
        scales = torch.zeros((npages, kv, page), device="cuda")
        if case["op"] != "cache":  # keys as the k norm leaves them, values of unit variance
            step = max(1, (1 << 26) // (kv * page * hd))
            for i in range(0, npages, step):
                x = randn(min(step, npages - i), kv, page, hd)
                c, s = _codes(_unit(x) if name == "k" else x, kind)
                codes[i:i + step].view(torch.int8).copy_(c.view(torch.int8))
                scales[i:i + step] = s
        st[name + "c"], st[name + "s"] = codes, scales
    total = int(ends[-1])
    if case["op"] == "cache":  # the fused rows of a layer's q, k and v products
        st["rows"] = torch.cat([_unit(randn(total, kv, hd)).reshape(total, kv * hd),
                                randn(total, kv * hd)], 1)
        st["k"], st["v"] = torch.empty((2, total, kv * hd), device="cuda").unbind(0)
    else:  # queries as the q norm leaves them, times what makes some keys count more than others
        st["q"] = (_unit(randn(total, case["heads"], hd)) * 2.5).reshape(total, -1)
        st["out"] = torch.empty_like(st["q"])
    if own:
        gemma_hip, gh = _lib()
        st["cache"] = gemma_hip.cache(st["kc"], st["vc"], st["ks"], st["vs"],
                                      gemma_hip.CACHE_I8 if kind == I8 else gemma_hip.CACHE_E4M3,
                                      npages, page, kv, hd)
        st["batch"] = gemma_hip.batch(st["table"], st["len"], st["row0"], batch, width, total,
                                      max(rows), max(lens))
        if case["op"] != "cache":
            n = gh.cache_attention_work(st["cache"], st["batch"], case["heads"], case["slide"],
                                        shared * page)
            st["work"] = torch.empty(max(1, n), dtype=torch.uint8, device="cuda")
    return st


# ---- one pass ------------------------------------------------------------------


def _plain_sample(st):
    l, t = st["logits"], st["t"].double()[:, None]
    v = l.shape[1]
    ordered, index = torch.sort(l, dim=1, descending=True, stable=True)
    far = ordered.double() - ordered[:, :1].double()
    w = torch.where(t > 0, torch.exp(far / torch.where(t > 0, t, 1.0)),
                    (torch.arange(v, device=l.device) == 0).double())
    total = torch.cumsum(w, 1)
    k = torch.where(st["k"] > 0, st["k"].long().clamp(max=v), v)[:, None]
    at_least = st["p"].double()[:, None] * total.gather(1, k - 1)
    n_p = torch.where(st["p"][:, None] < 1, (total < at_least).sum(1, keepdim=True) + 1, v)
    n_m = (w >= st["m"].double()[:, None]).sum(1, keepdim=True)
    n = torch.minimum(torch.minimum(k, n_p), n_m).clamp(min=1)
    kept = total.gather(1, n - 1)
    j = (total <= st["u"].double()[:, None] * kept).sum(1, keepdim=True)
    j = torch.minimum(j, n - 1)
    return dict(tokens=index.gather(1, j)[:, 0].int(),
                probs=(w.gather(1, j) / kept)[:, 0].float())


def _where(st):
    """Page and offset of every new row."""
    page = st["case"]["page"]
    return st["table"][st["seq"], st["pos"] // page].long(), st["pos"] % page


def _plain_cache(st):
    c = st["case"]
    kv, hd = c["kv"], c["hdim"]
    page, off = _where(st)
    out = {}
    for i, name in enumerate("kv"):
        x = st["rows"][:, i * kv * hd:(i + 1) * kv * hd].reshape(-1, kv, hd)
        codes, scales = _codes(x, c["type"])
        st[name + "c"].view(torch.int8)[page, :, off] = codes.view(torch.int8)
        st[name + "s"][page, :, off] = scales
        back = st[name + "c"].view(torch.int8)[page, :, off].view(st[name + "c"].dtype)
        out[name] = (back.float() * st[name + "s"][page, :, off][..., None]).reshape(-1, kv * hd)
    return out


def _gather(st, name, b, n, dtype):
    """The first n keys or values of sequence b, [kv][n][hdim]."""
    page = st["case"]["page"]
    pages = st["table"][b, :-(-n // page)].long()
    codes = st[name + "c"].view(torch.int8)[pages].view(st[name + "c"].dtype)
    x = codes.to(dtype) * st[name + "s"][pages][..., None].to(dtype)
    return x.transpose(0, 1).reshape(x.shape[1], -1, x.shape[3])[:, :n]


def _plain_attention(st):
    c = st["case"]
    heads, kv, hd, cap = c["heads"], c["kv"], c["hdim"], c["cap"]
    out, r = [], 0
    for b, (n, ln) in enumerate(zip(*st["seqs"])):
        first = max(0, ln - n + 1 - c["slide"]) if c["slide"] else 0
        k, v = (_gather(st, x, b, ln, torch.float32)[:, first:] for x in "kv")
        q = st["q"][r:r + n].reshape(n, kv, heads // kv, hd).permute(1, 2, 0, 3)
        s = torch.matmul(q.reshape(kv, -1, hd), k.transpose(1, 2).contiguous()) / math.sqrt(hd)
        if cap:
            s = torch.tanh(s / cap) * cap
        at = torch.arange(ln - n, ln, device=s.device)[:, None]
        key = torch.arange(first, ln, device=s.device)[None, :]
        off = key > at
        if c["slide"]:
            off = off | (key <= at - c["slide"])
        s = s.reshape(kv, heads // kv, n, -1).masked_fill(off, -math.inf)
        e = torch.exp(s - s.amax(-1, keepdim=True))
        o = torch.matmul(e.reshape(kv, -1, ln - first), v) / e.sum(-1).reshape(kv, -1, 1)
        out.append(o.reshape(kv, heads // kv, n, hd).permute(2, 0, 1, 3).reshape(n, heads * hd))
        r += n
    return torch.cat(out)


def run(st):
    c = st["case"]
    op = c["op"]
    if not own:
        return (_plain_sample if op == "sample" else _plain_cache if op == "cache"
                else _plain_attention)(st)
    gh = _lib()[1]
    s = torch.cuda.current_stream().cuda_stream
    if op == "sample":
        gh.sample(st["tokens"], st["probs"], st["logits"], c["vocab"], c["rows"], c["vocab"],
                  st["settings"], st["u"], st["work"], s)
        return dict(tokens=st["tokens"], probs=st["probs"])
    if op == "cache":
        w = c["kv"] * c["hdim"]
        gh.cache_write(st["cache"], st["batch"], st["rows"], 2 * w, st["rows"][:, w:], 2 * w, s)
        gh.cache_read(st["cache"], st["batch"], st["k"], w, st["v"], w, s)
        return dict(k=st["k"], v=st["v"])
    gh.cache_attention(st["out"], st["q"], c["heads"] * c["hdim"], st["cache"], st["batch"],
                       c["heads"], c["slide"], 1.0 / math.sqrt(c["hdim"]), c["cap"], False,
                       c.get("shared", 0) // c["page"] * c["page"], st["work"], s)
    return st["out"]


# ---- what a pass cannot do without ------------------------------------------------


def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return dict(bytes=4 * n + 28 * case["rows"], flops=2 * n)
    kv, hd = case["kv"], case["hdim"]
    rows, lens = _sequences(case)
    row = 2 * kv * (hd + 4)  # a position's keys and values
    table = 4 * case["batch"] * (2 + -(-max(lens) // case["page"]))
    if case["op"] == "cache":
        n = sum(rows)
        return dict(bytes=n * (2 * 8 * kv * hd + 2 * row) + table, flops=6 * n * kv * hd)
    seen = _seen(case)
    pairs = sum(hi - lo + 1 for s in seen for lo, hi in s)
    shared = case.get("shared", 0) // case["page"] * case["page"]
    first = min(s[0][0] for s in seen)
    keys = max(0, shared - first) + sum(s[-1][1] + 1 - max(s[0][0], shared) for s in seen)
    return dict(bytes=8 * sum(rows) * case["heads"] * hd + keys * row + table,
                flops=4 * case["heads"] * hd * pairs)


# ---- the same in 64 bits -----------------------------------------------------------


def _exact_sample(st):
    tokens, probs = [], []
    logits = st["logits"].double().cpu().numpy()
    t, k, p, m, u = (st[f].double().cpu().numpy() for f in "tkpmu")
    for i, l in enumerate(logits):
        order = np.argsort(-l, kind="stable")
        if t[i] == 0:
            tokens.append(order[0])
            probs.append(1.0)
            continue
        w = np.exp((l[order] - l[order[0]]) / t[i])
        if k[i] > 0:
            w = w[:int(k[i])]
        if p[i] < 1:
            run_ = np.cumsum(w)
            w = w[:np.searchsorted(run_, p[i] * run_[-1]) + 1]
        w = w[:max(1, int((w >= m[i]).sum()))]
        run_ = np.cumsum(w)
        j = min(int(np.searchsorted(run_, u[i] * run_[-1], side="right")), len(w) - 1)
        tokens.append(order[j])
        probs.append(w[j] / run_[-1])
    return dict(tokens=torch.tensor(np.array(tokens, np.int32)), probs=torch.tensor(probs))


def _exact_cache(st):
    c = st["case"]
    kv, hd, top = c["kv"], c["hdim"], TOP[c["type"]]
    out = {}
    for i, name in enumerate("kv"):
        x = st["rows"][:, i * kv * hd:(i + 1) * kv * hd].double().reshape(-1, hd)
        amax = x.abs().max(1, keepdim=True).values
        # the two roundings of the definition, to fp32, before the code's own
        y = (x * (top / amax).float().double()).float().double()
        if c["type"] == I8:
            code = torch.sign(y) * torch.floor((y.abs().float() + 0.5).double())
        else:  # steps of 2^(e - 3), of 2^-9 below 2^-6, halves to even
            step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
            code = torch.round(y / step) * step
        out[name] = (code * amax / top).reshape(-1, kv * hd)
    return out


def _exact_attention(st):
    c = st["case"]
    heads, hd, group = c["heads"], c["hdim"], c["heads"] // c["kv"]
    out, r = [], 0
    for b, (n, ln) in enumerate(zip(*st["seqs"])):
        k, v = (_gather(st, x, b, ln, torch.float64) for x in "kv")
        pos = ln - n + torch.arange(n, device="cuda").reshape(n, 1)
        key = torch.arange(ln, device="cuda").reshape(1, ln)
        seen = (key <= pos) & ((key > pos - c["slide"]) if c["slide"] else (key >= 0))
        for h in range(heads):
            s = st["q"][r:r + n, h * hd:(h + 1) * hd].double() @ k[h // group].t() * hd ** -0.5
            if c["cap"]:
                s = c["cap"] * torch.tanh(s / c["cap"])
            out.append(torch.softmax(torch.where(seen, s, -math.inf), 1) @ v[h // group])
        r += n
    out = [torch.cat(out[i:i + heads], 1) for i in range(0, len(out), heads)]
    return torch.cat(out)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(st)
    return _exact_cache(st) if case["op"] == "cache" else _exact_attention(st)
