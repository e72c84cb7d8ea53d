"""The operators between the products of a served batch, as timed cases.

A server's layer is more than its products and its attention, and its answers
more than the tokens drawn.  Each case is one pass through one of these:

    rope      heads turned by their positions, as they are or after their norm
    append    a batch's new rows through the q and k norms and the rotation: the
              queries out, keys and values into their sequences' 8-bit pages (and
              read back from them)
    norm      the norm behind a block, its gate and scales, the residual sum and the
              next block's norm, quantised for the next product or not
    adapters  the low-rank adapters of many requests, added to what a shared
              projection gave
    logprobs  log probabilities and ranks of given tokens, the rows' entropies and
              most likely tokens

With `own` false a pass computes the operator in elementary torch operations,
with `own` true by the library (gemma_hip.GemmaHip).  Widths are those of the
configurations in model_bin.

The formulas.  rope: x, or x / sqrt(mean x^2 + eps) (w + 1); pair j of the first `rot`
values of a head ((j, j + rot/2), or (2j, 2j+1)) turns by pos f_j, times an amplitude;
the others stay.  Angles and values in 64 bits, one rounding to fp32 at the end.
append: q and k so, rounded to fp32; k and v to codes and a scale per head (int8: scale =
amax (1/127), code = x (127/amax) to nearest, halves away from zero; e4m3: the same with
448, ties to even; every operation one fp32 rounding, rows of zeros with scale 0).
norm: x' = cx x + cy g N(y), rounded to fp32, h = N'(x'); N divides by the root of the
mean square plus eps and multiplies by w + 1, or takes the mean off first and applies w
and b; h is rounded to fp32, and made codes as above with scale 1 for rows of zeros.
adapters: dst = base + s_a (x A_a^T) B_a^T, a the adapter of the row's request, if any.
logprobs: p = softmax(l / T); log p of the given tokens, their ranks (1 and how many have
a larger logit, or an equal one and a lower index), -sum p log p, and the first n tokens
by falling logit, ties by rising index.
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
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6


def listed():
    return [
        # the queries of one decode step of eight gemma-3-1b sequences: the smallest, all latency
        dict(name="rope_step_1b", op="rope", rows=8, heads=4, hdim=256, rot=256, layout="half",
             norm=False, far=1001, scaling="none"),
        # a long prompt's heads, half of each turning in pairs of neighbours, positions up to 131072
        dict(name="rope_prompt_part", op="rope", rows=4096, heads=8, hdim=256, rot=128,
             layout="pairs", norm=True, far=131072, scaling="yarn"),
        # a decode step of eight gemma-3-1b sequences in a sliding layer
        dict(name="append_step_1b", op="append", batch=8, rows=1, ragged=False, len=1001, heads=4,
             kv=1, hdim=256, page=16, rot=256, layout="half", norm=True, scaling="none", type=I8),
        # a decode step of 64 gemma-3-4b sequences in a global layer, far positions at an eighth
        dict(name="append_step_4b_64", op="append", batch=64, rows=1, ragged=True, len=32768,
             heads=8, kv=4, hdim=256, page=64, rot=256, layout="half", norm=True,
             scaling="linear", type=E4M3),
        # four prompts of different lengths into a layer of gemma-3-4b, bandwidth
        dict(name="append_prompts_4b", op="append", batch=4, rows=4096, ragged=True, len=4096,
             heads=8, kv=4, hdim=256, page=64, rot=256, layout="half", norm=True, scaling="none",
             type=I8),
        # one token between two blocks of gemma-3-1b, codes for the next product
        dict(name="norm_step_1b", op="norm", rows=1, dim=1152, kind="rms", gate=False, quant=True),
        # a prompt between two blocks of gemma-3-4b
        dict(name="norm_prompt_4b", op="norm", rows=4096, dim=2560, kind="rms", gate=False,
             quant=False),
        # a decode step of 32 gemma-3-1b requests with 8 adapters between them, on q|k|v
        dict(name="adapters_step_1b_32", op="adapters", batch=32, rows=1, ragged=False, k=1152,
             n="1024 256 256", rank=16, count=8, type="bf16"),
        # a step's and a prompt chunk's rows of gemma-3-4b on gate|up, wide adapters
        dict(name="adapters_chunk_4b", op="adapters", batch=3, rows=613, ragged=True, k=2560,
             n="10240 10240", rank=64, count=2, type="f16"),
        # four prompts of different requests on gemma-3-4b's q|k|v
        dict(name="adapters_prompts_4b", op="adapters", batch=4, rows=1024, ragged=False, k=2560,
             n="2048 1024 1024", rank=16, count=4, type="bf16"),
        # one sampled token with 20 alternatives
        dict(name="logprobs_1", op="logprobs", rows=1, vocab=262144, spread=2.5, temperature=0.8,
             targets=1, top=20),
        # a chunk of a prompt scored, five alternatives each
        dict(name="logprobs_prompt_256", op="logprobs", rows=256, vocab=262144, spread=3.0,
             temperature=1.0, targets=1, top=5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "append", "append", "norm", "norm", "adapters", "adapters",
                     "logprobs", "logprobs"])
    turn = dict(layout=rng.choice(["half", "pairs"]), norm=rng.random() < 0.7,
                scaling=rng.choice(["none", "linear", "ntk", "bands", "yarn"]))
    if op == "rope":
        hdim = rng.choice([64, 72, 96, 128, 256])
        heads = rng.randint(1, 16)
        return dict(turn, op=op, rows=_log(rng, 1, max(1, 8388608 // (heads * hdim))), heads=heads,
                    hdim=hdim, rot=rng.choice([hdim, hdim // 8 * 4]),
                    far=_log(rng, 16, 131072))
    if op == "append":
        heads, kv, hdim = rng.choice([(4, 1, 256), (8, 4, 256), (4, 2, 128), (2, 2, 128)])
        rows = _log(rng, 1, 4096)
        batch = _log(rng, 1, max(1, min(64, 10000 // rows)))
        return dict(turn, op=op, heads=heads, kv=kv, hdim=hdim, rot=rng.choice([hdim, hdim // 2]),
                    page=rng.choice([16, 32, 64, 256]), type=rng.choice([I8, E4M3]), batch=batch,
                    rows=rows, ragged=batch > 1 and rng.random() < 0.6,
                    len=rows + rng.choice([0, _log(rng, 1, 30000 // batch)]))
    if op == "norm":
        dim = rng.choice([208, 256, 512, 640, 704, 1152, 2560])
        return dict(op=op, rows=_log(rng, 1, 10485760 // dim), dim=dim,
                    kind=rng.choice(["rms", "rms", "layer", "first"]), gate=rng.random() < 0.4,
                    quant=rng.random() < 0.6)
    if op == "adapters":
        k, n = rng.choice([(640, "1024 256 256"), (1152, "1024 256 256"), (1152, "6912 6912"),
                           (6912, "1152"), (1024, "1152"), (2560, "2048 1024 1024"),
                           (208, "1040 1040")])
        rows = rng.choice([1, 1, _log(rng, 2, 1024)])
        return dict(op=op, batch=_log(rng, 1, max(1, min(64, 2048 // rows))), rows=rows,
                    ragged=rows > 1 and rng.random() < 0.6, k=k, n=n, rank=rng.choice([8, 16, 32, 64]),
                    count=_log(rng, 1, 16), type=rng.choice(["bf16", "bf16", "f16", "f32"]))
    vocab = rng.choice([262144, _log(rng, 1000, 262144)])
    return dict(op=op, rows=_log(rng, 1, max(1, min(4096, (1 << 26) // vocab))), vocab=vocab,
                spread=round(rng.uniform(0.5, 5.0), 2), temperature=rng.choice([0.0, 0.7, 1.0, 1.5]),
                targets=rng.choice([1, 1, 1, 0, rng.randint(2, 8)]),
                top=rng.choice([0, 1, 5, 20, rng.randint(2, 64)]))


# ---- a case's sequences --------------------------------------------------------


def _sequences(case):
    """New rows and length of every sequence: about a quarter of `rows` to `rows`, or of a
    step's lengths, in no order, where they are ragged."""
    b, n, ln = case["batch"], case["rows"], case.get("len", case["rows"])
    share = [0.25 + 0.75 * ((i * 0.6180339887) % 1.0) if case["ragged"] else 1.0 for i in range(b)]
    if n == 1:
        return [1] * b, [max(1, int(ln * s)) for s in share]
    rows = [max(1, int(n * s)) for s in share]
    return rows, [r + ln - n for r in rows]


def _widths(case):
    """The outputs of the projections side by side."""
    return [int(n) for n in case["n"].split()]


def _freqs(rot, theta, scaling):
    """Radians a position of each pair, and the amplitude."""
    f = theta ** (-2.0 * np.arange(rot // 2) / rot)
    if scaling == "none":
        return f, 1.0
    if scaling == "linear":
        return f / 8.0, 1.0
    if scaling == "ntk":
        return (theta * 8.0 ** (rot / (rot - 2.0))) ** (-2.0 * np.arange(rot // 2) / rot), 1.0
    if scaling == "bands":
        factor, low, high, before = 8.0, 1.0, 4.0, 8192.0
        turns = before * f / (2 * math.pi)
        s = np.clip((turns - low) / (high - low), 0.0, 1.0)
        return f * ((1 - s) / factor + s), 1.0
    factor, fast, slow, before = 16.0, 32.0, 1.0, 8192.0

    def dim(turns):
        return rot * math.log(before / (turns * 2 * math.pi)) / (2 * math.log(theta))

    lo, hi = max(0, math.floor(dim(fast))), min(rot - 1, math.ceil(dim(slow)))
    s = np.clip((np.arange(rot // 2) - lo) / max(hi - lo, 0.001), 0.0, 1.0)
    return f * (s / factor + 1 - s), 0.1 * math.log(factor) + 1.0


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


def _rotary(st):
    c, gemma_hip = st["case"], _lib()[0]
    kind = gemma_hip.ROPE_HALF if c["layout"] == "half" else gemma_hip.ROPE_PAIRS
    return gemma_hip.rotary(st["freq"], c["rot"], kind, st["amp"])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    host = np.random.default_rng(seed)

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    st = dict(case=dict(case))
    return globals()["_prepare_" + case["op"]](case, st, randn, g, host)


def _turns(case, st):
    theta = 10000.0 if case["scaling"] == "none" else 1e6
    f, amp = _freqs(case["rot"], theta, case["scaling"])
    st.update(freq=torch.tensor(f, dtype=torch.float64, device="cuda"),
              amp=float(np.float32(amp)))


def _prepare_rope(case, st, randn, g, host):
    rows, heads, hd = case["rows"], case["heads"], case["hdim"]
    _turns(case, st)
    st.update(x=randn(rows, heads * hd), w=randn(hd) * 0.1 if case["norm"] else None,
              pos=torch.tensor(host.integers(0, case["far"], rows), dtype=torch.int32, device="cuda"))
    if own:
        st.update(out=torch.empty_like(st["x"]), rotary=_rotary(st))
    return st


def _prepare_append(case, st, randn, g, host):
    kv, hd, page, heads, batch = (case[f] for f in ("kv", "hdim", "page", "heads", "batch"))
    rows, lens = _sequences(case)
    need = [-(-ln // page) for ln in lens]
    width, npages = max(need), sum(need)
    table = np.zeros((batch, width), np.int32)
    order, at = host.permutation(npages).astype(np.int32), 0
    for b in range(batch):
        table[b, :need[b]] = order[at:at + need[b]]
        at += need[b]
    ends = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    total = int(ends[-1])
    _turns(case, st)
    dtype = torch.int8 if case["type"] == I8 else torch.float8_e4m3fn
    st.update(
        table=torch.tensor(table, device="cuda"), row0=torch.tensor(ends, device="cuda"),
        len=torch.tensor(lens, dtype=torch.int32, device="cuda"),
        pos=torch.tensor(np.concatenate([np.arange(ln - n, ln) for n, ln in zip(rows, lens)]),
                         device="cuda"),
        seq=torch.tensor(np.repeat(np.arange(batch), rows), device="cuda"),
        x=randn(total, (heads + 2 * kv) * hd),  # a layer's q | k | v products
        wq=randn(hd) * 0.1 if case["norm"] else None, wk=randn(hd) * 0.1 if case["norm"] else None)
    for name in "kv":
        st[name + "c"] = torch.zeros((npages, kv, page, hd), dtype=torch.int8,
                                     device="cuda").view(dtype)
        st[name + "s"] = torch.zeros((npages, kv, page), device="cuda")
    if own:
        gemma_hip, gh = _lib()
        q, k, v = heads * hd, kv * hd, kv * hd
        st.update(q=torch.empty((total, q), device="cuda"), k=torch.empty((total, k), device="cuda"),
                  v=torch.empty((total, v), device="cuda"))
        st["cache"] = gemma_hip.cache(st["kc"], st["vc"], st["ks"], st["vs"],
                                      gemma_hip.CACHE_I8 if case["type"] == I8
                                      else gemma_hip.CACHE_E4M3, npages, page, kv, hd)
        st["batch"] = gemma_hip.batch(st["table"], st["len"], st["row0"], batch, width, total,
                                      max(rows), max(lens))
        x, n = st["x"], q + k + v
        st["heads"] = gemma_hip.heads(x, n, x[:, q:], n, x[:, q + k:], n, st["q"], 0, heads,
                                      st["wq"], st["wk"], EPS, _rotary(st))
    return st


def _prepare_norm(case, st, randn, g, host):
    rows, dim = case["rows"], case["dim"]
    st.update(x=randn(rows, dim) * 3.0, y=randn(rows, dim), w=randn(dim) * 0.1,
              w0=randn(dim) * 0.1, b=randn(dim) * 0.1, cx=1.0, cy=1.0,
              g=randn(rows, dim) if case["gate"] else None)
    if case["gate"]:
        st.update(cx=0.5, cy=1.25)
    if own:
        gemma_hip, gh = _lib()
        x_out, h = torch.empty((2, rows, dim), device="cuda").unbind(0)
        st.update(x_out=x_out, h=h, hq=torch.empty((rows, dim), dtype=torch.int8, device="cuda"),
                  hs=torch.empty(rows, device="cuda"))
        rms = [gemma_hip.norm(gemma_hip.NORM_RMS, st[w], None, 1.0, EPS) for w in ("w0", "w")]
        if case["kind"] == "layer":  # a block of its own norm only
            after, before = None, gemma_hip.norm(gemma_hip.NORM_LAYER, st["w"], st["b"], 0.0, EPS)
        else:
            after, before = rms if case["kind"] == "rms" else (None, rms[1])
        st["spec"] = gemma_hip.residual(
            x=st["x"], y=st["y"], gate=st["g"], x_scale=st["cx"], y_scale=st["cy"], after=after,
            before=before, x_out=x_out, h=None if case["quant"] else h,
            hq=st["hq"] if case["quant"] else None, hs=st["hs"] if case["quant"] else None)
    return st


def _prepare_adapters(case, st, randn, g, host):
    rows, _ = _sequences(case)
    ns = _widths(case)
    k, rank, count, batch = (case[f] for f in ("k", "rank", "count", "batch"))
    total, dtype = sum(rows), TYPES[case["type"]]
    ends = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    ids = host.integers(-1 if batch > 4 else 0, count, batch).astype(np.int32)  # some have none
    st.update(ids=torch.tensor(ids, device="cuda"), row0=torch.tensor(ends, device="cuda"),
              seq=torch.tensor(np.repeat(np.arange(batch), rows), device="cuda"),
              scale=torch.rand(count, generator=g, device="cuda") + 0.5,
              x=randn(total, k), base=randn(total, sum(ns)),
              a=[(randn(count, rank, k) / math.sqrt(k)).to(dtype) for _ in ns],
              b=[(randn(count, n, rank) / math.sqrt(rank)).to(dtype) for n in ns])
    if own:
        gemma_hip, gh = _lib()
        kind = getattr(gemma_hip, "ADAPTER_" + case["type"].upper())
        st["out"] = torch.empty_like(st["base"])
        st["ad"] = gemma_hip.adapters(st["row0"], st["ids"], st["scale"], batch, total, max(rows),
                                      count, rank, kind)
        st["jobs"] = gemma_hip.adapter_jobs(list(zip(st["a"], st["b"], ns)))
        st["work"] = torch.empty(max(1, gh.adapters_work(st["ad"], len(ns), k)), dtype=torch.uint8,
                                 device="cuda")
    return st


def _prepare_logprobs(case, st, randn, g, host):
    rows, vocab, nt, top = case["rows"], case["vocab"], case["targets"], case["top"]
    st.update(logits=randn(rows, vocab) * case["spread"],
              t=torch.full((rows,), case["temperature"], device="cuda"),
              ids=torch.tensor(host.integers(0, vocab, (rows, nt)), dtype=torch.int32, device="cuda"))
    if nt:  # what was said is mostly what was likely
        likely = st["logits"].argmax(1).int()
        st["ids"][::2, 0] = likely[::2]
    if own:
        gemma_hip, gh = _lib()
        st["out"] = dict(logp=torch.empty((rows, nt), device="cuda"),
                         rank=torch.empty((rows, nt), dtype=torch.int32, device="cuda"),
                         entropy=torch.empty(rows, device="cuda"),
                         top=torch.empty((rows, top), dtype=torch.int32, device="cuda"),
                         top_logp=torch.empty((rows, top), device="cuda"))
        st["scores"] = gemma_hip.scores(**st["out"])
        st["work"] = torch.empty(max(1, gh.logprobs_work(rows, vocab, nt, top)), dtype=torch.uint8,
                                 device="cuda")
    return st


# ---- one pass, plain -------------------------------------------------------------


def _codes(x, kind, zero=0.0):
    """Codes (as the type that holds them) and scales of rows x; zero: the scale of zeros."""
    amax = x.abs().amax(-1)
    inv = torch.where(amax > 0, (TOP[kind] / amax.double()), 1.0).float()
    scale = amax * torch.tensor(1.0 / TOP[kind], dtype=torch.float32, device=x.device)
    scale = torch.where(amax > 0, scale, zero)
    y = x * inv[..., None]
    if kind == I8:
        return torch.trunc(y + torch.copysign(torch.full_like(y, 0.5), y)).to(torch.int8), scale
    return y.clamp(-TOP[kind], TOP[kind]).to(torch.float8_e4m3fn), scale


def _plain_turn(x, w, pos, freq, amp, c):
    """Heads x [rows][heads][hdim], in 64 bits, as the next step's codes lie next to borders."""
    x = x.double()
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * (w.double() + 1.0)
    rot, n = c["rot"], c["rot"] // 2
    angle = pos.double()[:, None] * freq
    cos, sin = (torch.cos(angle) * amp)[:, None], (torch.sin(angle) * amp)[:, None]
    first, second = (slice(0, n), slice(n, rot)) if c["layout"] == "half" else \
        (slice(0, rot, 2), slice(1, rot, 2))
    out = x.clone()
    out[..., first] = x[..., first] * cos - x[..., second] * sin
    out[..., second] = x[..., second] * cos + x[..., first] * sin
    return out.float()


def _plain_rope(st):
    c = st["case"]
    x = st["x"].reshape(c["rows"], c["heads"], c["hdim"])
    return _plain_turn(x, st["w"], st["pos"], st["freq"], st["amp"], c).reshape(c["rows"], -1)


def _split(st):
    c = st["case"]
    q, k = c["heads"] * c["hdim"], c["kv"] * c["hdim"]
    return [st["x"][:, a:b].reshape(st["x"].shape[0], -1, c["hdim"])
            for a, b in ((0, q), (q, q + k), (q + k, q + 2 * k))]


def _plain_append(st):
    c = st["case"]
    total = st["x"].shape[0]
    q, k, v = _split(st)
    q = _plain_turn(q, st["wq"], st["pos"], st["freq"], st["amp"], c)
    k = _plain_turn(k, st["wk"], st["pos"], st["freq"], st["amp"], c)
    page = st["table"][st["seq"], st["pos"] // c["page"]].long()
    off = st["pos"] % c["page"]
    out = dict(q=q.reshape(total, -1))
    for name, x in (("k", k), ("v", v)):
        codes, scales = _codes(x, c["type"])
        st[name + "c"].view(torch.int8)[page, :, off] = codes.view(torch.int8)
        st[name + "s"][page, :, off] = scales
        back = st[name + "c"].view(torch.int8)[page, :, off].view(st[name + "c"].dtype)
        out[name] = (back.float() * st[name + "s"][page, :, off][..., None]).reshape(total, -1)
    return out


def _plain_rms(x, w):
    return x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * (w.double() + 1.0)


def _plain_norm(st):
    c = st["case"]
    y = st["y"].double()  # 64 bits: the codes lie next to borders
    if c["kind"] == "rms":
        y = _plain_rms(y, st["w0"])
    y = y * st["cy"]
    if st["g"] is not None:
        y = y * st["g"]
    x = (st["x"].double() * st["cx"] + y).float()
    h = x.double()
    if c["kind"] == "layer":
        h = h - h.mean(-1, keepdim=True)
        h = h / (h.square().mean(-1, keepdim=True) + EPS).sqrt() * st["w"] + st["b"]
    else:
        h = _plain_rms(h, st["w"])
    h = h.float()
    if c["quant"]:
        codes, scales = _codes(h, I8, 1.0)
        h = codes * scales[:, None]
    return dict(x=x, h=h)


def _plain_adapters(st):
    """All adapters' first halves for every row, the other adapters' results made zeros."""
    c = st["case"]
    ids = st["ids"][st["seq"]].long()
    one = (ids[:, None] == torch.arange(c["count"], device=ids.device)) * st["scale"]
    out = []
    for a, b in zip(st["a"], st["b"]):
        u = st["x"] @ a.float().reshape(-1, c["k"]).t()
        u = u.reshape(-1, c["count"], c["rank"]) * one[..., None]
        out.append(u.reshape(-1, c["count"] * c["rank"]) @
                   b.float().permute(0, 2, 1).reshape(c["count"] * c["rank"], -1))
    return st["base"] + torch.cat(out, 1)


def _plain_logprobs(st):
    c = st["case"]
    l, ids = st["logits"], st["ids"].long()
    rows, vocab = l.shape
    top = l.amax(1, keepdim=True)
    given = l.gather(1, ids)
    index = torch.arange(vocab, device=l.device)
    rank = [1 + ((l > given[:, j:j + 1]) | ((l == given[:, j:j + 1]) & (index < ids[:, j:j + 1])))
            .sum(1) for j in range(c["targets"])]
    rank = torch.stack(rank, 1).int() if rank else ids.int()
    # by falling logit, then rising index: one whole number that orders so
    bits = l.view(torch.int32).long()
    key = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * (1 << 20) + ((1 << 20) - 1 - index)
    best = (1 << 20) - 1 - (torch.topk(key, c["top"], dim=1).values & ((1 << 20) - 1))
    if c["temperature"] == 0.0:  # all on the first of the largest
        first = ((1 << 20) - 1 - (key.amax(1) & ((1 << 20) - 1)))[:, None]
        zero = torch.zeros((), device=l.device)
        return dict(logp=torch.where(ids == first, zero, -math.inf), rank=rank,
                    entropy=torch.zeros(rows, device=l.device), top=best.int(),
                    top_logp=torch.where(best == first, zero, -math.inf))
    d = (l - top) / st["t"][:, None]
    e = torch.exp(d)
    total = e.sum(1, dtype=torch.float64)
    log = torch.log(total)
    entropy = log - (e * d).sum(1, dtype=torch.float64) / total
    chosen = l.gather(1, best)
    t = st["t"].double()[:, None]
    return dict(logp=((given.double() - top) / t - log[:, None]).float(), rank=rank,
                entropy=entropy.float(), top=best.int(),
                top_logp=((chosen.double() - top) / t - log[:, None]).float())


# ---- one pass ------------------------------------------------------------------


def run(st):
    c = st["case"]
    op = c["op"]
    if not own:
        return globals()["_plain_" + op](st)
    gh = _lib()[1]
    s = torch.cuda.current_stream().cuda_stream
    if op == "rope":
        gh.rope(st["out"], 0, st["x"], 0, c["rows"], c["heads"], c["hdim"], st["pos"], st["w"],
                EPS, st["rotary"], s)
        return st["out"]
    if op == "append":
        gh.cache_append(st["cache"], st["batch"], st["heads"], s)
        gh.cache_read(st["cache"], st["batch"], st["k"], 0, st["v"], 0, s)
        return dict(q=st["q"], k=st["k"], v=st["v"])
    if op == "norm":
        gh.norm_residual(st["spec"], c["rows"], c["dim"], s)
        return dict(x=st["x_out"],
                    h=st["hq"] * st["hs"][:, None] if c["quant"] else st["h"])
    if op == "adapters":
        gh.adapters_add(st["out"], 0, st["base"], 0, st["ad"], st["jobs"], st["x"], 0, c["k"],
                        st["work"], s)
        return st["out"]
    gh.logprobs(st["scores"], st["logits"], 0, c["rows"], c["vocab"], st["t"], st["ids"],
                c["targets"], c["top"], st["work"], s)
    return st["out"]


# ---- what a pass cannot do without ------------------------------------------------


def work(case):
    op = case["op"]
    if op == "rope":
        n = case["rows"] * case["heads"] * case["hdim"]
        return dict(bytes=8 * n + 4 * case["rows"] + 4 * case["rot"], flops=8 * n)
    if op == "append":
        kv, hd, heads = case["kv"], case["hdim"], case["heads"]
        rows, lens = _sequences(case)
        n = sum(rows)
        codes = 2 * kv * (hd + 4)  # a position's keys and values
        # q | k | v read, q written, codes written, and read back as fp32
        one = 4 * (2 * heads + 2 * kv) * hd + codes + codes + 8 * kv * hd
        table = 4 * case["batch"] * (2 + -(-max(lens) // case["page"]))
        return dict(bytes=n * one + table, flops=n * hd * (8 * heads + 16 * kv))
    if op == "norm":
        n = case["rows"] * case["dim"]
        # x and y (and the gate) read, x' and h written, h's codes made values
        h = (1 + 1 + 4) if case["quant"] else 4
        return dict(bytes=n * (12 + (4 if case["gate"] else 0) + h) + 12 * case["dim"], flops=12 * n)
    if op == "adapters":
        n, jobs, total = sum(_widths(case)), len(_widths(case)), sum(_sequences(case)[0])
        size = 4 if case["type"] == "f32" else 2
        used = min(case["count"], case["batch"])
        return dict(bytes=4 * total * (case["k"] + 2 * n) +
                    used * case["rank"] * size * (case["k"] * jobs + n),
                    flops=2 * total * case["rank"] * (case["k"] * jobs + n))
    n = case["rows"] * case["vocab"]
    return dict(bytes=4 * n + case["rows"] * (8 + 12 * case["targets"] + 8 * case["top"]),
                flops=6 * n)


# ---- the same in 64 bits -----------------------------------------------------------


def _exact_turn(st, x, w):
    """Pair by pair as a product of complex numbers."""
    c = st["case"]
    rows, heads, hd, rot = *x.shape, c["rot"]
    x = x.double()
    if w is not None:
        x = x * torch.rsqrt(torch.linalg.vector_norm(x, dim=-1, keepdim=True) ** 2 / hd + EPS)
        x = x + x * w.double()
    part = x[..., :rot]
    part = part.reshape(rows, heads, 2, rot // 2).transpose(2, 3) if c["layout"] == "half" else \
        part.reshape(rows, heads, rot // 2, 2)
    angle = (st["pos"].double().reshape(rows, 1) * st["freq"]).reshape(rows, 1, rot // 2)
    turned = torch.view_as_real(torch.view_as_complex(part.contiguous()) *
                                torch.polar(torch.full_like(angle, st["amp"]), angle))
    if c["layout"] == "half":
        turned = turned.transpose(2, 3)
    return torch.cat([turned.reshape(rows, heads, rot), x[..., rot:]], -1)


def _exact_codes(x, kind):
    """Values of the codes of rows x that are fp32, by the definition's own roundings."""
    top = TOP[kind]
    x = x.double()
    amax = x.abs().max(-1, keepdim=True).values
    y = (x * torch.nan_to_num(top / amax, posinf=1.0).float().double()).float().double()
    if kind == I8:
        code = torch.sign(y) * torch.floor((y.abs().float() + 0.5).double())
    else:  # steps of 2^(e - 3), of 2^-9 below 2^-6, halves to even
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
        code = torch.round(y / step) * step
    return code * amax / top


def _exact_append(st):
    total = st["x"].shape[0]
    q, k, v = _split(st)
    kind = st["case"]["type"]
    return dict(q=_exact_turn(st, q, st["wq"]).reshape(total, -1),
                k=_exact_codes(_exact_turn(st, k, st["wk"]).float(), kind).reshape(total, -1),
                v=_exact_codes(v, kind).reshape(total, -1))


def _exact_norm(st):
    c = st["case"]

    def scaled(v, mean, mul, add):
        v = v - mean
        return v * ((v ** 2).sum(1, keepdim=True) / c["dim"] + EPS) ** -0.5 * mul + add

    y = st["y"].double()
    if c["kind"] == "rms":
        y = scaled(y, 0.0, 1.0 + st["w0"].double(), 0.0)
    g = st["g"].double() if st["g"] is not None else 1.0
    x = st["cx"] * st["x"].double() + st["cy"] * g * y
    r = x.float().double()
    if c["kind"] == "layer":
        h = scaled(r, r.sum(1, keepdim=True) / c["dim"], st["w"].double(), st["b"].double())
    else:
        h = scaled(r, 0.0, 1.0 + st["w"].double(), 0.0)
    return dict(x=x, h=_exact_codes(h.float(), I8) if c["quant"] else h)


def _exact_adapters(st):
    """Request by request."""
    c, out = st["case"], st["base"].double()
    ends = st["row0"].tolist()
    for i, a in enumerate(st["ids"].tolist()):
        if a < 0:
            continue
        rows, at = slice(ends[i], ends[i + 1]), 0
        for n, first, second in zip(_widths(c), st["a"], st["b"]):
            u = torch.mm(st["x"][rows].double(), first[a].double().t())
            out[rows, at:at + n] += st["scale"][a].double() * torch.mm(u, second[a].double().t())
            at += n
    return out


def _exact_logprobs(st):
    """Row by row, on sorted values."""
    c = st["case"]
    logp, entropy, top_logp = [], [], []
    for l, ids, t in zip(st["logits"], st["ids"].long(), st["t"].double()):
        ordered, order = torch.sort(l, descending=True, stable=True)
        if t == 0:
            p = torch.full_like(l, -math.inf, dtype=torch.float64)
            p[order[0]] = 0.0
            entropy.append(torch.zeros((), dtype=torch.float64, device=l.device))
        else:
            p = torch.log_softmax(l.double() / t, 0)
            entropy.append(-(p.exp() * p).sum())
        logp.append(p[ids])
        top_logp.append(p[order[:c["top"]]])
    return dict(logp=torch.stack(logp), rank=None, entropy=torch.stack(entropy), top=None,
                top_logp=torch.stack(top_logp))


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "rope":
        x = st["x"].reshape(case["rows"], case["heads"], case["hdim"])
        return _exact_turn(st, x, st["w"]).reshape(case["rows"], -1)
    return globals()["_exact_" + op](st)
