"""The operators of serving a batch of sequences, one by one and together: the
8-bit paged key/value cache (gemma_hip_cache_write, _read), attention over it
(gemma_hip_cache_attention, its shared prefix included) and sampling
(gemma_hip_sample), against plain numpy in 64 bits.

Bars.  Codes, scales and read values follow a definition of single fp32 roundings:
equal to the bit.  Tokens: equal (a weight in a sum is off by at most 2^-39 of itself,
and a random number falls that close to a border once in 10^8 draws).
Attention, relative to the largest |v| that a row sees: scores up to about 10 are
fp32 sums whose 16 or so roundings leave 1e-6, which is the weights' relative error
and at most that of the output, and the value sums' own roundings leave about as
much; ten times both is 2e-5, also the bar of the fp32-cache kernels."""

from __future__ import annotations

import ctypes
import os
import subprocess
import threading

import numpy as np
import pytest

import gemma_hip
from gemma_hip import CACHE_E4M3, CACHE_I8

F32, F64 = np.float32, np.float64
ATT_TOL = 2e-5
TOP = {CACHE_I8: 127.0, CACHE_E4M3: 448.0}
KINDS = {"i8": CACHE_I8, "e4m3": CACHE_E4M3}
CSRC = os.path.join(gemma_hip.PKG_DIR, "csrc")


# ---- the definitions, in numpy ------------------------------------------------


def e4m3_table():
    """The 256 values of e4m3 codes (0x7f and 0xff are NaN)."""
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    v = np.where((c & 127) == 127, np.nan, v)
    return np.where(c & 128, -v, v)


E4M3 = e4m3_table()


def to_e4m3(y):
    """Codes of finite fp32 values within +-448, ties to even."""
    a = np.abs(y.astype(F64))
    step = 2.0 ** (np.floor(np.log2(np.maximum(a, 2.0 ** -6))) - 3)
    a = np.rint(a / step) * step
    code = np.searchsorted(E4M3[:127], a)
    assert np.array_equal(E4M3[code], a)
    return (code + 128 * np.signbit(y)).astype(np.uint8)


def quantise(x, kind):
    """Codes (uint8) and scales of rows x [..., hdim] fp32."""
    amax = np.abs(x).max(-1)
    bad = ~np.isfinite(x).all(-1)
    with np.errstate(all="ignore"):
        scale = amax * F32(1.0 / TOP[kind])
        inv = (TOP[kind] / amax.astype(F64)).astype(F32)
        y = (x * inv[..., None]).astype(F32)
        if kind == CACHE_I8:
            code = np.trunc(y + np.copysign(F32(0.5), y))
            code = np.where(np.isfinite(code), code, 0).astype(np.int8).view(np.uint8)
        else:
            code = to_e4m3(np.clip(np.nan_to_num(y), -448, 448))
    zero = bad | (amax == 0)
    return (np.where(zero[..., None], 0, code).astype(np.uint8),
            np.where(bad, np.nan, scale).astype(F32))


def values(code, scale, kind):
    v = code.view(np.int8).astype(F32) if kind == CACHE_I8 else E4M3[code].astype(F32)
    return v * scale[..., None]


def attend(q, k, v, pos, length, slide, asc, cap, dense):
    """One row and head in 64 bits: q [hdim] over k, v [len][hdim], and the largest
    |v| it sees."""
    hi = -1 if pos < 0 else length - 1 if dense else pos
    lo = max(0, pos + 1 - slide) if slide and not dense else 0
    keys = [i for i in range(lo, hi + 1) if not np.isinf(k[i]).any()]  # inf: not there
    if not keys:
        return np.zeros(q.shape, F64), 0.0
    s = k[keys].astype(F64) @ q.astype(F64) * asc
    if cap:
        s = np.tanh(s / cap) * cap
    p = np.exp(s - s.max())
    return p @ v[keys].astype(F64) / p.sum(), float(np.abs(v[keys]).max())


def near(x):
    """The least |x| but for zeros: what is equal is so in exact arithmetic too."""
    x = np.abs(x[x != 0])
    return float(x.min()) if len(x) else 1.0


def draw_token(l, t, k, p, m, u):
    """(token, probability, margin) of one row: how far, in shares of the kept sum,
    the draw and the cuts are from falling on another token."""
    l = np.where(np.isnan(l), -np.inf, l.astype(F64))
    order = np.argsort(-l, kind="stable")
    order = order[l[order] > -np.inf]
    if len(order) == 0:
        return -1, 0.0, 1.0
    if not t > 0:
        return int(order[0]), 1.0, 1.0
    top = l[order[0]]
    w = np.where(l[order] == top, 1.0, 0.0) if np.isinf(top) else np.exp((l[order] - top) / t)
    margin = 1.0
    if k > 0:
        w = w[:k]
    if p < 1:
        c = np.cumsum(w)
        n = min(int(np.searchsorted(c, p * c[-1])) + 1, len(w))
        margin = near(c - p * c[-1]) / c[-1] if p > 0 else 1.0
        w = w[:n]
    if m > 0:
        margin = min(margin, near(w - m))
        w = w[:max(1, int((w >= m).sum()))]
    c = np.cumsum(w)
    j = min(int(np.searchsorted(c, u * c[-1], side="right")), len(w) - 1)
    if u > 0:
        margin = min(margin, near(c[:-1] - u * c[-1]) / c[-1])
    return int(order[j]), w[j] / c[-1], margin


# ---- the definitions themselves -------------------------------------------------


def test_e4m3_matches_torch():
    import torch

    t = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(t, E4M3, equal_nan=True)
    y = np.concatenate([np.linspace(-448, 448, 4001), np.linspace(-0.05, 0.05, 2001),
                        2.0 ** -np.arange(0, 14)]).astype(F32)
    c = torch.from_numpy(y).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(E4M3[c], E4M3[to_e4m3(y)])


def test_quantise_is_gemma_hip_quantize(oracle):
    x = np.random.default_rng(0).standard_normal((40, 256)).astype(F32)
    q, s = oracle.quantize_acts(x)
    code, scale = quantise(x, CACHE_I8)
    assert np.array_equal(code.view(np.int8), q) and np.array_equal(scale, s)


def test_reference_catches_planted_mistakes():
    """A window off by one, no cap, the wrong scale, one key more: all far past the
    bar; another order among equals, a filter left out: another token."""
    rng = np.random.default_rng(1)
    q, k, v = (rng.standard_normal(s).astype(F32) for s in ((128,), (60, 128), (60, 128)))
    asc = 128 ** -0.5
    want, vmax = attend(q, k, v, 50, 60, 16, asc, 30.0, False)
    for other in ((50, 60, 17, asc, 30.0, False), (50, 60, 16, asc, 0.0, False),
                  (50, 60, 16, asc * asc, 30.0, False), (51, 60, 16, asc, 30.0, False),
                  (50, 60, 16, asc, 30.0, True)):
        got, _ = attend(q, k, v, *other)
        assert np.abs(got - want).max() > 10 * ATT_TOL * vmax, other
    l = np.array([1.0, 3.0, 3.0, 2.0])
    assert draw_token(l, 1.0, 1, 1.0, 0.0, 0.9)[0] == 1
    assert draw_token(l, 1.0, 2, 1.0, 0.0, 0.9)[0] == 2
    assert draw_token(l, 1.0, 0, 1.0, 0.0, 0.9)[0] == 3
    assert draw_token(l, 1.0, 0, 0.6, 0.0, 0.9)[0] == 2
    assert draw_token(l, 1.0, 0, 1.0, 0.5, 0.9)[0] == 2
    assert draw_token(l, 0.0, 0, 1.0, 0.0, 0.9)[0] == 1


# ---- tables and refusals, without a GPU ------------------------------------------


@pytest.fixture(scope="session")
def tables(tmp_path_factory):
    """kv_cache.h's functions, compiled for the host."""
    d = tmp_path_factory.mktemp("kv")
    src = d / "kv.cpp"
    src.write_text('#include "kv_cache.h"\n'
                   'using namespace gh;\n'
                   'extern "C" {\n'
                   'void seq(KvBatch *b, int i, int *o) { KvSeq s = kv_seq(*b, i);'
                   ' o[0] = s.r0; o[1] = s.n; o[2] = s.len; }\n'
                   'long slot(KvCache *c, KvBatch *b, int i, int p, int h)'
                   ' { return kv_slot(*c, *b, i, p, h); }\n'
                   'int find(int *r, int n, int x) { return kv_find(r, n, x); }\n'
                   'void span(int p, int l, int s, int d, int *o)'
                   ' { KvSpan x = kv_span(p, l, s, d); o[0] = x.lo; o[1] = x.hi; }\n'
                   '}\n')
    so = d / "kv.so"
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-std=c++17", "-I", CSRC, str(src), "-o",
                    str(so)], check=True)
    lib = ctypes.CDLL(str(so))
    lib.slot.restype = ctypes.c_long
    return lib


class HostCache(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("k", "v", "ks", "vs")] + \
               [(n, ctypes.c_int) for n in ("type", "npages", "shift", "nkv", "hdim")]


class HostBatch(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("pages", "len", "row0")] + \
               [(n, ctypes.c_int) for n in ("batch", "width", "rows", "max_rows", "max_len")]


def test_tables_stay_in_bounds(tables):
    """Whatever the device tables hold, rows, lengths and slots stay inside."""
    rng = np.random.default_rng(2)
    for _ in range(300):
        n, width, shift, nkv = (int(rng.integers(1, h)) for h in (6, 5, 7, 4))
        shift += 3
        npages, rows = int(rng.integers(1, 9)), int(rng.integers(0, 40))
        max_rows, max_len = int(rng.integers(0, rows + 1)), int(rng.integers(0, (width << shift) + 1))
        wild = rng.random() < 0.5
        pages = rng.integers(-3, npages + 3, (n, width)).astype(np.int32)
        ln = rng.integers(-5, 2 * max_len + 5, n).astype(np.int32)
        row0 = rng.integers(-4, rows + 9, n + 1).astype(np.int32)
        if wild:
            pages[0, 0], ln[0], row0[0] = -2 ** 31, 2 ** 31 - 1, 2 ** 31 - 1
        else:
            row0.sort()
        b = HostBatch(pages.ctypes.data, ln.ctypes.data, row0.ctypes.data, n, width, rows,
                      max_rows, max_len)
        c = HostCache(None, None, None, None, 0, npages, shift, nkv, 128)
        for i in range(n):
            o = (ctypes.c_int * 3)()
            tables.seq(ctypes.byref(b), i, o)
            assert 0 <= o[0] and 0 <= o[1] <= max_rows and o[0] + o[1] <= rows
            assert 0 <= o[2] <= max_len
            for p in range(0, max_len, max(1, max_len // 7)):
                at = tables.slot(ctypes.byref(c), ctypes.byref(b), i, p, nkv - 1)
                page = pages[i, p >> shift]
                if 0 <= page < npages:
                    assert at == ((int(page) * nkv + nkv - 1) << shift) + p % (1 << shift)
                    assert at < npages * nkv << shift
                else:
                    assert at == -1
        for r in range(-2, rows + 12):
            f = tables.find(row0.ctypes.data_as(ctypes.c_void_p), n, r)
            assert -1 <= f < n
            if not wild:
                own = [i for i in range(n) if row0[i] <= r < row0[i + 1]]
                assert f == (own[0] if own else -1)


def test_slots_pass_32_bits(tables):
    pages = np.array([[2 ** 31 - 2]], np.int32)
    b = HostBatch(pages.ctypes.data, None, None, 1, 1, 1, 1, 256)
    c = HostCache(None, None, None, None, 0, 2 ** 31 - 1, 8, 3, 256)
    assert tables.slot(ctypes.byref(c), ctypes.byref(b), 0, 255, 2) == \
        (((2 ** 31 - 2) * 3 + 2) << 8) + 255


def test_spans(tables):
    o = (ctypes.c_int * 2)()
    for p in range(-2, 9):
        for ln in range(max(p + 1, 0), 10):
            for slide in (0, 1, 4, 20):
                for dense in (0, 1):
                    tables.span(p, ln, slide, dense, o)
                    want = [] if p < 0 else list(range(ln)) if dense else \
                        [k for k in range(p + 1) if not slide or k > p - slide]
                    assert list(range(o[0], o[1] + 1)) == want


def fake(n=4096):
    """An address that passes for device memory where nothing is run."""
    return 0x7f0000000000 + n


def good():
    c = gemma_hip.cache(fake(), fake(), fake(), fake(), CACHE_I8, 8, 16, 2, 128)
    b = gemma_hip.batch(fake(), fake(), fake(), 2, 4, 5, 4, 64)
    return c, b


BAD = [  # field of the cache or batch, value, a word of the message
    ("c", "type", 7, "type"), ("c", "hdim", 64, "heads of 64"), ("c", "nkv", 0, "heads"),
    ("c", "page", 24, "power of two"), ("c", "page", 8, "power of two"),
    ("c", "npages", 0, "pages"), ("c", "k", None, "null"), ("c", "vs", None, "null"),
    ("c", "v", fake(8), "aligned"), ("c", "ks", fake(4), "aligned"),
    ("b", "batch", -1, "batch"), ("b", "batch", 70000, "batch"), ("b", "rows", -1, "batch"),
    ("b", "max_rows", 6, "batch"), ("b", "max_len", 65, "batch"), ("b", "max_len", -1, "batch"),
    ("b", "pages", None, "null"), ("b", "len", None, "null"), ("b", "row0", None, "null"),
]


@pytest.mark.parametrize("what,field,value,word", BAD)
def test_bad_caches_and_batches_are_refused(what, field, value, word):
    lib = gemma_hip.load()
    c, b = good()
    setattr(c if what == "c" else b, field, value)
    calls = {
        "write": lambda: lib.gemma_hip_cache_write(c, b, fake(), 256, fake(), 256, None),
        "read": lambda: lib.gemma_hip_cache_read(c, b, fake(), 256, fake(), 256, None),
        "attention": lambda: lib.gemma_hip_cache_attention(
            fake(), fake(), 512, c, b, 4, 0, 1.0, 0.0, 0, 0, None, 0, None),
    }
    for name, call in calls.items():
        assert call() == 1, name
        msg = lib.gemma_hip_last_error().decode()
        assert name in msg and word in msg, msg
    if word not in ("null", "aligned"):
        assert lib.gemma_hip_cache_attention_work(c, b, 4, 0, 0) == ctypes.c_size_t(-1).value


def test_more_rows_than_the_kernels_count_are_refused():
    lib = gemma_hip.load()
    c, b = good()
    b.rows = b.max_rows = 1 << 26
    assert lib.gemma_hip_cache_write(c, b, fake(), 256, fake(), 256, None) == 1
    assert "too many rows" in lib.gemma_hip_last_error().decode()
    b.max_rows = 1  # few of each sequence, but the shared prefix is read by all of them
    assert lib.gemma_hip_cache_attention(fake(), fake(), 512, c, b, 4, 0, 1.0, 0.0, 0, 0, None, 0,
                                         None) == 1
    assert "too many rows" in lib.gemma_hip_last_error().decode()
    assert lib.gemma_hip_cache_attention_work(c, b, 4, 0, 0) == ctypes.c_size_t(-1).value


def test_bad_rows_and_settings_are_refused():
    lib = gemma_hip.load()
    c, b = good()
    rows = [((fake(), 255, fake(), 256), "multiple of 4"), ((fake(), 252, fake(), 256), "stride"),
            ((fake(), 256, fake(4), 256), "aligned"), ((None, 256, fake(), 256), "null")]
    for args, word in rows:
        for call in (lib.gemma_hip_cache_write, lib.gemma_hip_cache_read):
            assert call(c, b, *args, None) == 1
            assert word in lib.gemma_hip_last_error().decode()

    def attention(out=fake(), q=fake(), qs=512, heads=4, slide=0, shared=0):
        return lib.gemma_hip_cache_attention(out, q, qs, c, b, heads, slide, 1.0, 0.0, 0, shared,
                                             None, 0, None)

    for kw, word in ((dict(out=None), "out"), (dict(out=fake(4)), "out"), (dict(q=None), "null"),
                     (dict(q=fake(8)), "aligned"), (dict(qs=508), "stride"),
                     (dict(heads=3), "heads"), (dict(heads=0), "heads"), (dict(slide=-1), "window"),
                     (dict(shared=-1), "prefix"), (dict(shared=65), "prefix")):
        assert attention(**kw) == 1
        assert word in lib.gemma_hip_last_error().decode(), kw
    assert lib.gemma_hip_cache_write(None, b, fake(), 0, fake(), 0, None) == 1
    assert lib.gemma_hip_cache_read(c, None, fake(), 0, fake(), 0, None) == 1

    def sample(tokens=fake(), logits=fake(), stride=0, rows=2, vocab=100, u=fake()):
        return lib.gemma_hip_sample(tokens, None, logits, stride, rows, vocab, None, u, None, 0,
                                    None)

    for kw, word in ((dict(tokens=None), "null"), (dict(logits=None), "null"),
                     (dict(u=None), "null"), (dict(stride=99), "stride"), (dict(rows=-1), "shape"),
                     (dict(vocab=0), "shape"), (dict(vocab=524289), "shape"),
                     (dict(rows=65536), "shape")):
        assert sample(**kw) == 1
        assert word in lib.gemma_hip_last_error().decode(), kw
    assert lib.gemma_hip_sample_work(1, 0) == ctypes.c_size_t(-1).value


# ---- a batch on the GPU ------------------------------------------------------------


def cuda(a):
    import torch

    return torch.from_numpy(np.array(a, order="C")).cuda()


class Paged:
    """A cache on the GPU whose spare places hold what must never be read: NaN
    scales and, in e4m3, the codes of NaN."""

    def __init__(self, seqs, kv, hd, page, kind, rng, shared=0, spare=2, width=None):
        self.seqs, self.kv, self.hd, self.page, self.kind = seqs, kv, hd, page, kind
        self.n = [n for n, _ in seqs]
        self.len = [ln for _, ln in seqs]
        batch = len(seqs)
        need = [-(-ln // page) for ln in self.len]
        whole = shared // page
        self.width = max(need + [1]) if width is None else width
        total = whole + sum(max(0, x - whole) for x in need) + spare
        ids = rng.permutation(total).astype(np.int32)
        self.table = np.full((batch, self.width), -7, np.int32)
        at = whole
        for b in range(batch):
            self.table[b, :min(whole, need[b])] = ids[:min(whole, need[b])]
            more = max(0, need[b] - whole)
            self.table[b, whole:whole + more] = ids[at:at + more]
            at += more
        self.spare = ids[at:]
        code = 0x7f
        self.codes = {x: np.full((total, kv, page, hd), code, np.uint8) for x in "kv"}
        self.scales = {x: np.full((total, kv, page), np.nan, F32) for x in "kv"}
        self.row0 = np.concatenate([[0], np.cumsum(self.n)]).astype(np.int32)
        self.rows = int(self.row0[-1])

    def put(self, b, pos, x, h, name):
        code, scale = quantise(x[None], self.kind)
        page = self.table[b, pos // self.page]
        if 0 <= page < self.codes["k"].shape[0]:
            self.codes[name][page, h, pos % self.page] = code[0]
            self.scales[name][page, h, pos % self.page] = scale[0]

    def fill(self, rng, scale=1.0, upto=None):
        """Random values at every position (below its end less `upto` rows)."""
        for b, ln in enumerate(self.len):
            last = ln if upto is None else ln - upto[b]
            for pos in range(0, max(0, last), self.page):
                m = min(self.page, last - pos)
                page = self.table[b, pos // self.page]
                for name in "kv":
                    code, sc = quantise((rng.standard_normal((self.kv, m, self.hd)) * scale)
                                        .astype(F32), self.kind)
                    self.codes[name][page, :, :m], self.scales[name][page, :, :m] = code, sc

    def seq_values(self, b, name, h):
        """Values of a sequence's positions, inf where there is no page."""
        out = np.full((self.len[b], self.hd), np.inf, F32)
        for pos in range(0, self.len[b], self.page):
            page = self.table[b, pos // self.page]
            if 0 <= page < self.codes["k"].shape[0]:
                m = min(self.page, self.len[b] - pos)
                out[pos:pos + m] = values(self.codes[name][page, h, :m],
                                          self.scales[name][page, h, :m], self.kind)
        return out

    def device(self):
        self.d = {x: (cuda(self.codes[x]), cuda(self.scales[x])) for x in "kv"}
        self.tab, self.dlen, self.drow0 = (cuda(np.asarray(a, np.int32)) for a in
                                           (self.table, self.len, self.row0))
        npages = self.codes["k"].shape[0]
        c = gemma_hip.cache(self.d["k"][0], self.d["v"][0], self.d["k"][1], self.d["v"][1],
                            self.kind, npages, self.page, self.kv, self.hd)
        return c

    def batch(self, rows=None, max_rows=None, max_len=None):
        return gemma_hip.batch(self.tab, self.dlen, self.drow0, len(self.seqs), self.width,
                               self.rows if rows is None else rows,
                               max(self.n + [0]) if max_rows is None else max_rows,
                               max(self.len + [0]) if max_len is None else max_len)


def stream():
    import torch

    return torch.cuda.current_stream().cuda_stream


WRITES = {  # sequences (new rows, positions), kv heads, head dim, page
    "steps": ([(1, 1), (1, 17), (1, 16), (1, 100)], 1, 256, 16),
    "prompts": ([(33, 33), (5, 70), (0, 12), (128, 131), (1, 1), (0, 0)], 4, 256, 32),
    "hd128": ([(19, 40), (64, 64), (1, 65)], 3, 128, 64),
    "one_page": ([(7, 300)], 2, 128, 512),
    "many": ([(i % 3, 3 + i % 40) for i in range(100)] + [(90, 100), (0, 7), (3, 60)], 1, 128, 16),
    "ahead": ([(5, 3), (2, 2)], 2, 256, 16),  # rows before position 0: nowhere
}


@pytest.mark.gpu
@pytest.mark.parametrize("kind", sorted(KINDS))
@pytest.mark.parametrize("case", sorted(WRITES))
def test_write_and_read_back(gh, case, kind):
    import torch

    seqs, kv, hd, page = WRITES[case]
    kind = KINDS[kind]
    rng = np.random.default_rng(len(case) + kind)
    p = Paged(seqs, kv, hd, page, kind, rng)
    p.fill(rng, upto=p.n)
    c = p.device()
    more = 3  # rows behind the last sequence's
    stride = 3 * kv * hd + 8
    x = rng.standard_normal((p.rows + more, stride)).astype(F32)
    if p.rows > 3:
        x[0, :hd] = 0.0                       # a row of zeros
        x[1, hd // 2] *= 1e4                  # an outlier
        x[2, :hd] *= 1e-30                    # small ones
        x[3, :hd] = rng.integers(-5, 6, hd)   # ties and equal magnitudes
    ks, vs = x[:, :kv * hd], x[:, kv * hd + 4:2 * kv * hd + 4]
    dx = cuda(x)
    gh.cache_write(c, p.batch(p.rows + more), dx, stride, dx[:, kv * hd + 4:], stride, stream())
    for b, (n, ln) in enumerate(seqs):
        for i in range(n):
            pos, r = ln - n + i, p.row0[b] + i
            for h in range(kv):
                if pos >= 0:
                    p.put(b, pos, ks[r, h * hd:(h + 1) * hd], h, "k")
                    p.put(b, pos, vs[r, h * hd:(h + 1) * hd], h, "v")
    back = [torch.full((p.rows + more, kv * hd + 4), 5.0, device="cuda") for _ in "kv"]
    gh.cache_read(c, p.batch(p.rows + more), back[0], kv * hd + 4, back[1], kv * hd + 4, stream())
    torch.cuda.synchronize()
    for i, name in enumerate("kv"):
        code, scale = (t.cpu().numpy() for t in p.d[name])
        assert np.array_equal(code, p.codes[name]), name  # every other place as it was
        assert np.array_equal(scale, p.scales[name], equal_nan=True), name
        want = np.full((p.rows + more, kv * hd + 4), 5.0, F32)
        for b, (n, ln) in enumerate(seqs):
            for r in range(n):
                pos = ln - n + r
                for h in range(kv):
                    at = slice(h * hd, (h + 1) * hd)
                    want[p.row0[b] + r, at] = p.seq_values(b, name, h)[pos] if pos >= 0 else 0.0
        assert np.array_equal(back[i].cpu().numpy(), want), name


@pytest.mark.gpu
@pytest.mark.parametrize("kind", sorted(KINDS))
def test_rows_that_are_not_finite(gh, kind):
    """They read back as NaN, their codes stay finite, and rows that don't see them
    are as if they weren't there."""
    import torch

    kind, rng = KINDS[kind], np.random.default_rng(5)
    p = Paged([(40, 40)], 1, 128, 16, kind, rng)
    c = p.device()
    x = rng.standard_normal((40, 128)).astype(F32)
    y = rng.standard_normal((40, 128)).astype(F32)
    bad_k, bad_v = x.copy(), y.copy()
    bad_k[20, 3], bad_v[25, 7], bad_v[33, 9] = np.nan, np.inf, -np.inf
    q = rng.standard_normal((40, 128)).astype(F32)
    out = []
    for k, v in ((x, y), (bad_k, bad_v)):
        gh.cache_write(c, p.batch(), cuda(k), 0, cuda(v), 0, stream())
        o, rk, rv = (torch.empty((40, 128), device="cuda") for _ in range(3))
        gh.cache_read(c, p.batch(), rk, 0, rv, 0, stream())
        gh.cache_attention(o, cuda(q), 0, c, p.batch(), 1, 8, 0.1, 0.0, False, 0, None, stream())
        torch.cuda.synchronize()
        out.append([t.cpu().numpy() for t in (o, rk, rv)])
    (o0, k0, v0), (o1, k1, v1) = out
    assert np.isnan(k1[20]).all() and np.isnan(v1[[25, 33]]).all()
    keep = [i for i in range(40) if i not in (20, 25, 33)]
    assert np.array_equal(k1[keep], k0[keep]) and np.array_equal(v1[keep], v0[keep])
    codes = p.d["v"][0].cpu().numpy()[p.table[0, :3], 0].reshape(48, 128)[:40]
    assert not codes[[25, 33]].any()
    assert kind == CACHE_I8 or not np.isin(codes, [0x7f, 0xff]).any()
    sees = {i for b in (20, 25, 33) for i in range(b, min(40, b + 8))}  # the window is 8
    for i in range(40):
        if i in sees:
            assert np.isnan(o1[i]).all(), i
        else:
            assert np.array_equal(o1[i], o0[i]), i


# sequences (new rows, positions), heads, kv, head dim, page, window, cap, dense, shared
ATTN = {
    "one_token": ([(1, 1)], 4, 1, 256, 16, 0, 0.0, False, 0),
    "step": ([(1, 1), (1, 16), (1, 17), (1, 33), (1, 250)], 4, 1, 256, 16, 0, 0.0, False, 0),
    "step_4b": ([(1, 100), (1, 40), (1, 129)], 8, 4, 256, 64, 0, 0.0, False, 0),
    "step_window": ([(1, 100), (1, 40), (1, 700), (1, 16)], 4, 1, 256, 32, 50, 0.0, False, 0),
    "step_cap": ([(1, 77), (1, 300)], 4, 2, 128, 16, 0, 5.0, False, 0),
    "step_no_gqa": ([(1, 60), (1, 61)], 3, 3, 128, 16, 0, 0.0, False, 0),
    "step_wide": ([(1, 90), (1, 31)], 32, 1, 128, 16, 0, 0.0, False, 0),
    "wide_prefix": ([(1, 90), (3, 131), (0, 70), (1, 64)], 32, 1, 128, 16, 0, 0.0, False, 64),
    "widest": ([(1, 40), (2, 33)], 1024, 1, 128, 16, 0, 0.0, False, 0),
    "widest_prefix": ([(1, 40), (1, 33)], 1024, 2, 128, 16, 20, 0.0, False, 32),
    "step_24": ([(1, 90), (1, 31)], 24, 2, 256, 16, 0, 0.0, False, 0),
    "few_rows": ([(3, 90), (2, 31), (4, 4)], 4, 1, 256, 16, 0, 0.0, False, 0),
    "prompt": ([(70, 70)], 4, 1, 256, 16, 0, 0.0, False, 0),
    "many_mixed": ([(i % 3, 3 + i % 40) for i in range(70)] + [(90, 100), (0, 7), (40, 300)] +
                   [(1 + i % 7, 80 + i) for i in range(60)], 4, 1, 256, 16, 0, 0.0, False, 0),
    "many_prompts": ([(17 + i % 9, 30 + i) for i in range(67)] + [(0, 0), (70, 900)], 4, 2, 128, 16,
                     0, 0.0, False, 0),
    "prompt_behind": ([(45, 200), (7, 130)], 8, 4, 256, 64, 0, 0.0, False, 0),
    "prompt_window": ([(130, 220)], 4, 2, 128, 32, 33, 0.0, False, 0),
    "prompt_window_1": ([(40, 50)], 4, 2, 128, 32, 1, 0.0, False, 0),
    "prompt_cap": ([(65, 100)], 4, 1, 256, 32, 0, 50.0, False, 0),
    "dense": ([(64, 80), (20, 20), (1, 50)], 4, 1, 256, 16, 8, 0.0, True, 0),
    "mixed": ([(1, 300), (50, 60), (0, 20), (1, 1), (17, 400), (0, 0), (3, 200)], 4, 1, 256, 16, 0,
              0.0, False, 0),
    "mixed_4b": ([(1, 90), (70, 170), (2, 2), (1, 65)], 8, 4, 256, 16, 64, 0.0, False, 0),
    "ahead": ([(6, 4), (1, 0), (40, 30)], 4, 1, 128, 16, 0, 0.0, False, 0),
    "prefix": ([(1, 150), (1, 129), (1, 200), (1, 131)], 4, 1, 256, 16, 0, 0.0, False, 128),
    "prefix_odd": ([(1, 150), (1, 121), (2, 200), (1, 140)], 8, 4, 256, 16, 0, 0.0, False, 112),
    "prefix_window": ([(1, 150), (1, 129), (3, 260)], 4, 2, 128, 16, 60, 0.0, False, 128),
    "prefix_prompt": ([(30, 150), (70, 260), (1, 97), (0, 100)], 4, 1, 256, 32, 0, 0.0, False, 96),
    "prefix_cap": ([(1, 150), (1, 97)], 4, 1, 256, 32, 0, 20.0, False, 96),
    "prefix_past_some": ([(1, 150), (1, 40), (2, 64), (1, 1)], 4, 1, 128, 16, 0, 0.0, False, 96),
    "prefix_all": ([(1, 96), (1, 96), (1, 96)], 4, 1, 128, 16, 0, 0.0, False, 96),
    "prefix_dense": ([(9, 150), (3, 100)], 4, 2, 128, 16, 0, 0.0, True, 64),
    "prefix_many": ([(1, 100 + 7 * i) for i in range(40)], 4, 1, 128, 16, 0, 0.0, False, 96),
}


def check_attention(gh, p, heads, slide, cap, dense, shared, asc, rng, q=None, qpad=8, work=None,
                    rows=None, step=1, max_len=None):
    """Runs the call and compares every row (or every step-th) with attend()."""
    import torch

    hd, kv = p.hd, p.kv
    rows = p.rows if rows is None else rows
    if q is None:
        q = rng.standard_normal((rows, heads * hd + qpad)).astype(F32)
    c = p.device()
    out = torch.full((rows, heads * hd), 3.0, device="cuda")
    gh.cache_attention(out, cuda(q), q.shape[1], c, p.batch(rows, max_len=max_len), heads, slide, asc,
                       cap, dense, shared, work, stream())
    torch.cuda.synchronize()
    got = out.cpu().numpy().reshape(rows, heads, hd)
    worst = 0.0
    for b, (n, ln) in enumerate(p.seqs):
        for h in range(heads):
            k, v = (p.seq_values(b, x, h // (heads // kv)) for x in "kv")
            for i in range(0, n, step):
                r = p.row0[b] + i
                want, vmax = attend(q[r, h * hd:(h + 1) * hd], k, v, ln - n + i, ln, slide, asc,
                                    cap, dense)
                if vmax == 0.0:
                    assert (got[r, h] == 0).all(), (b, i, h)
                    continue
                err = np.abs(got[r, h] - want).max() / vmax
                worst = max(worst, err)
                assert err <= ATT_TOL, (b, i, h, err)
    assert (got[p.rows:] == 3.0).all()  # rows behind the last sequence, as they were
    print(f"largest error / max |v|: {worst:.3g}", flush=True)
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("kind", sorted(KINDS))
@pytest.mark.parametrize("case", sorted(ATTN))
def test_attention(gh, case, kind):
    seqs, heads, kv, hd, page, slide, cap, dense, shared = ATTN[case]
    rng = np.random.default_rng(len(case) + 7 * KINDS[kind])
    p = Paged(seqs, kv, hd, page, KINDS[kind], rng, shared)
    p.fill(rng)
    check_attention(gh, p, heads, slide, cap, dense, shared, hd ** -0.5, rng, rows=p.rows + 2)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", sorted(KINDS))
@pytest.mark.parametrize("asc,amp", [(-0.08, 1.0), (0.0, 1.0), (0.05, 30.0), (1e-3, 1e3),
                                     (0.088, 1e-3)])
def test_attention_scales(gh, kind, asc, amp):
    """Negative, zero, large and small score scales; q and the cache far from 1."""
    rng = np.random.default_rng(11)
    p = Paged([(1, 90), (40, 70)], 2, 128, 16, KINDS[kind], rng)
    p.fill(rng, scale=0.01 if amp > 1 else 1.0)
    q = (rng.standard_normal((p.rows, 4 * 128)) * amp).astype(F32)
    check_attention(gh, p, 4, 0, 0.0, False, 0, asc, rng, q=q)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 30])
def test_attention_values_of_many_magnitudes(gh, rows):
    """Positions whose values lie 2^30 apart keep their own precision: a row that
    sees only small ones (window) is as exact, relative to them, as one that sees
    the large ones; zeros in between do no harm."""
    rng = np.random.default_rng(12)
    p = Paged([(rows, 200), (rows, 120)], 1, 128, 16, CACHE_I8, rng)
    p.fill(rng)
    for page in range(p.codes["v"].shape[0]):
        p.scales["v"][page] *= F32(2.0) ** rng.integers(-30, 1, p.scales["v"][page].shape)
    p.scales["v"][p.table[0, 11]] = 0.0
    p.codes["v"][p.table[0, 11]] = 0
    check_attention(gh, p, 4, 5, 0.0, False, 0, 0.05, rng)


@pytest.mark.gpu
def test_attention_bad_pages(gh):
    """Ids outside the cache stand for keys that aren't there: single pages, the
    last one, and all of a sequence's."""
    rng = np.random.default_rng(13)
    p = Paged([(1, 100), (1, 60), (30, 90), (2, 40)], 2, 128, 16, CACHE_E4M3, rng)
    p.fill(rng)
    p.table[0, 2], p.table[1, 3], p.table[2, 0] = -1, 2 ** 31 - 1, p.codes["k"].shape[0]
    p.table[3, :] = -2 ** 31
    check_attention(gh, p, 4, 0, 0.0, False, 0, 0.09, rng)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,kind", [(4, 1, "i8"), (8, 4, "e4m3")])
def test_attention_long(gh, heads, kv, kind):
    """Long caches, split over the keys, beside short ones."""
    rng = np.random.default_rng(14)
    p = Paged([(1, 20011), (1, 5), (1, 4096), (2, 9001)], kv, 256, 64, KINDS[kind], rng)
    p.fill(rng)
    check_attention(gh, p, heads, 0, 0.0, False, 0, 0.0625, rng)


@pytest.mark.gpu
def test_attention_long_prompt_and_prefix(gh):
    rng = np.random.default_rng(15)
    p = Paged([(300, 2500), (1, 2100), (9, 2049)], 1, 256, 64, CACHE_I8, rng, shared=2048)
    p.fill(rng)
    check_attention(gh, p, 4, 0, 0.0, False, 2048, 0.0625, rng, step=7)
    check_attention(gh, p, 4, 512, 0.0, False, 2048, 0.0625, rng, step=7)
    check_attention(gh, p, 4, 0, 0.0, False, 0, 0.0625, rng, step=7)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,hdim,kind,slide,cap,shared", [
    (4, 1, 256, "i8", 0, 0.0, 0), (4, 1, 256, "e4m3", 0, 30.0, 1200), (4, 1, 256, "i8", 1500, 0.0, 0),
    (4, 1, 256, "e4m3", 1501, 0.0, 1216), (4, 1, 256, "i8", 0, 0.0, 1296),
    (8, 2, 128, "i8", 0, 0.0, 1200), (8, 2, 128, "e4m3", 1500, 30.0, 0)])
def test_attention_many_rows_over_many_keys(gh, heads, kv, hdim, kind, slide, cap, shared):
    """Enough of both (more than 20 tiles of 32 keys by 64 query vectors for each of the
    card's 256 compute units) that a workgroup takes 128 vectors, prefixes included."""
    rng = np.random.default_rng(19)
    p = Paged([(1300, 2600), (1, 1390), (901, 1400), (0, 1300)], kv, hdim, 16, KINDS[kind], rng,
              shared=shared)
    p.fill(rng)
    check_attention(gh, p, heads, slide, cap, False, shared, 0.0625, rng, step=53)


@pytest.mark.gpu
@pytest.mark.parametrize("hdim,kind", [(128, "e4m3"), (256, "i8")])
def test_attention_prefix_beside_long_or_many_sequences(gh, hdim, kind):
    """Single tokens behind a prefix in launches of their own: one with more than 64 tiles of
    keys of its own, and more than 512 sequences by key/value heads."""
    rng = np.random.default_rng(21)
    p = Paged([(1, 3500), (2, 1300), (1, 900), (0, 1100), (1, 1025)], 1, hdim, 32, KINDS[kind],
              rng, shared=1024)
    p.fill(rng)
    check_attention(gh, p, 4, 0, 0.0, False, 1024, 0.0625, rng)
    check_attention(gh, p, 4, 700, 20.0, False, 1024, 0.0625, rng)
    p = Paged([(i % 3, 64 + i % 70) for i in range(301)], 2, hdim, 16, KINDS[kind], rng, shared=64)
    p.fill(rng)
    check_attention(gh, p, 4, 0, 0.0, False, 64, 0.0625, rng)


@pytest.mark.gpu
@pytest.mark.parametrize("slide,dense,shared", [(0, False, 0), (90, False, 0), (90, True, 0),
                                                (0, False, 64), (300, True, 64)])
def test_attention_lengths_far_below_their_bound(gh, slide, dense, shared):
    """As a captured step has them: the host knows that no sequence passes 131072."""
    rng = np.random.default_rng(22)
    p = Paged([(1, 700), (3, 130), (1, 66), (50, 400)], 1, 256, 64, CACHE_E4M3, rng, shared=shared,
              width=2048)
    p.fill(rng)
    check_attention(gh, p, 4, slide, 0.0, dense, shared, 0.0625, rng, max_len=131072)
    p = Paged([(1, 700), (3, 130), (1, 66)], 2, 128, 64, CACHE_I8, rng, shared=shared, width=2048)
    p.fill(rng)
    check_attention(gh, p, 4, slide, 0.0, dense, shared, 0.0625, rng, max_len=131072)


@pytest.mark.gpu
@pytest.mark.parametrize("hdim", [128, 256])
def test_rows_without_a_page_table(gh, hdim):
    """Sequences of rows and no positions need no pages: nothing is written, and what is
    read or attended to is zeros."""
    import torch

    p = Paged([(1, 20)], 1, hdim, 16, CACHE_I8, np.random.default_rng(20))
    c = p.device()
    for n in ([1, 1], [40, 1]):
        rows = sum(n)
        b = gemma_hip.batch(None, cuda(np.zeros(2, np.int32)),
                            cuda(np.array([0, n[0], rows], np.int32)), 2, 0, rows, max(n), 0)
        x = torch.randn(rows, 4 * hdim, device="cuda")
        k, v = torch.ones(rows, hdim, device="cuda"), torch.ones(rows, hdim, device="cuda")
        gh.cache_write(c, b, k, 0, v, 0, stream())
        gh.cache_read(c, b, k, 0, v, 0, stream())
        out = torch.ones(rows, 4 * hdim, device="cuda")
        gh.cache_attention(out, x, 0, c, b, 4, 0, 1.0, 0.0, False, 0, None, stream())
        torch.cuda.synchronize()
        assert not k.any() and not v.any() and not out.any()


@pytest.mark.gpu
def test_attention_tables_that_lie(gh):
    """Lengths and rows past what the host said are cut to it; nothing is written
    outside (the buffers' surroundings stay as they were)."""
    import torch

    rng = np.random.default_rng(16)
    p = Paged([(1, 64), (3, 64), (1, 64)], 1, 128, 16, CACHE_I8, rng)
    p.fill(rng)
    c = p.device()
    p.dlen.copy_(cuda(np.array([2 ** 31 - 1, -5, 64], np.int32)))
    p.drow0.copy_(cuda(np.array([0, 900, 2, 5], np.int32)))
    pad = 64
    whole = torch.full((p.rows + 2 * pad, 4 * 128), 3.0, device="cuda")
    q = torch.randn((p.rows, 4 * 128), device="cuda")
    kv = torch.randn((p.rows, 128), device="cuda")
    gh.cache_write(c, p.batch(max_rows=3), kv, 0, kv, 0, stream())
    gh.cache_attention(whole[pad:], q, 0, c, p.batch(max_rows=3), 4, 0, 0.1, 0.0, False, 16, None,
                       stream())
    gh.cache_read(c, p.batch(max_rows=3), whole[pad:, :128].contiguous(), 0, kv, 0, stream())
    torch.cuda.synchronize()
    got = whole.cpu().numpy()
    assert (got[:pad] == 3.0).all() and (got[pad + p.rows:] == 3.0).all()


@pytest.mark.gpu
def test_nothing_to_do(gh):
    rng = np.random.default_rng(17)
    p = Paged([(0, 0), (0, 20)], 1, 128, 16, CACHE_I8, rng)
    c = p.device()
    for b in (p.batch(), gemma_hip.batch(None, None, None, 0, 0, 0, 0, 0)):
        gh.cache_write(c, b, None, 0, None, 0, stream())
        gh.cache_read(c, b, None, 0, None, 0, stream())
        gh.cache_attention(None, None, 0, c, b, 4, 0, 1.0, 0.0, False, 0, None, stream())
        assert gh.cache_attention_work(c, b, 4, 0, 0) >= 0
    gh.sample(None, None, None, 0, 0, 100, None, None, None, stream())


# ---- sampling ------------------------------------------------------------------


def check_sample(gh, l, t=None, k=None, p=None, m=None, u=None, stride=None, work=None):
    import torch

    rows, vocab = l.shape
    rng = np.random.default_rng(rows * vocab)
    u = rng.random(rows).astype(F32) if u is None else np.asarray(u, F32)
    stride = vocab if stride is None else stride
    full = np.full((rows, stride), np.nan, F32)
    full[:, :vocab] = l
    if stride > vocab:
        full[:, vocab:] = 1e30  # columns that are none of the vocabulary's
    arr = [None if a is None else cuda(np.broadcast_to(np.asarray(a, d), (rows,)))
           for a, d in ((t, F32), (k, np.int32), (p, F32), (m, F32))]
    tokens = torch.full((rows + 1,), 77, dtype=torch.int32, device="cuda")
    probs = torch.full((rows + 1,), 77.0, device="cuda")
    gh.sample(tokens, probs, cuda(full), stride, rows, vocab, gemma_hip.sampling(*arr), cuda(u),
              work, stream())
    torch.cuda.synchronize()
    tokens, probs = tokens.cpu().numpy(), probs.cpu().numpy()
    assert tokens[rows] == 77 and probs[rows] == 77.0

    def at(a, i, default):
        return default if a is None else np.broadcast_to(np.asarray(a), (rows,))[i]

    for i in range(rows):
        tok, prob, margin = draw_token(l[i], F64(F32(at(t, i, 1.0))), int(at(k, i, 0)),
                                       F64(F32(at(p, i, 1.0))), F64(F32(at(m, i, 0.0))),
                                       F64(u[i]))
        if margin < 1e-9:
            continue  # on a border to the last bits: no token is wrong
        assert tokens[i] == tok, (i, tokens[i], tok, margin)
        # one rounding to fp32, and the weights' 2^-44
        assert abs(probs[i] - prob) <= 2.0 ** -24 * prob + 2.0 ** -40, (i, probs[i], prob)
    return tokens[:rows]


SAMPLES = {  # rows, vocabulary, spread, temperature, top-k, top-p, min-p
    "plain": (5, 1000, 2.0, None, None, None, None),
    "chat": (4, 262144, 3.0, 0.8, 64, 0.95, None),
    "flat": (2, 262144, 0.5, 2.0, None, 0.9, None),
    "flat_k": (2, 262144, 0.3, 1.0, 100000, 0.5, None),
    "peaked": (3, 32000, 30.0, 1.0, None, 0.99, None),
    "min_p": (4, 262143, 3.0, 1.0, None, None, 0.05),
    "all": (6, 50257, 2.0, 1.3, 500, 0.9, 0.01),
    "greedy": (3, 262144, 1.0, 0.0, 5, 0.5, 0.5),
    "k1": (3, 4097, 1.0, 1.0, 1, None, None),
    "p0": (3, 4097, 1.0, 1.0, None, 0.0, None),
    "m1": (3, 4097, 1.0, 1.0, None, None, 1.0),
    "one": (2, 1, 1.0, 0.7, 3, 0.9, 0.1),
    "two": (9, 2, 1.0, 0.7, None, None, None),
    "k_vocab": (2, 777, 1.0, 1.0, 777, None, None),
    "k_more": (2, 777, 1.0, 1.0, 100000, 0.9, None),
    "cold": (3, 30000, 2.0, 1e-4, None, 0.9, None),
    "hot": (3, 30000, 2.0, 1e6, None, 0.9, None),
    "largest": (1, 524288, 2.0, 1.0, 3000, 0.99, None),
}


@pytest.mark.gpu
@pytest.mark.parametrize("case", sorted(SAMPLES))
def test_sample(gh, case):
    rows, vocab, spread, t, k, p, m = SAMPLES[case]
    rng = np.random.default_rng(len(case) + vocab)
    l = (rng.standard_normal((rows, vocab)) * spread).astype(F32)
    check_sample(gh, l, t, k, p, m, stride=vocab + 5)
    check_sample(gh, l, t, k, p, m, u=np.zeros(rows))
    check_sample(gh, l, t, k, p, m, u=np.full(rows, 1 - 2.0 ** -24))


@pytest.mark.gpu
def test_sample_mixed_rows(gh):
    """Every row with settings of its own, odd ones among them."""
    rng = np.random.default_rng(21)
    rows, vocab = 64, 20011
    l = (rng.standard_normal((rows, vocab)) * rng.uniform(0.2, 8, (rows, 1))).astype(F32)
    t = rng.choice([0.0, -1.0, 0.3, 1.0, 1.7, np.nan, np.inf], rows)
    k = rng.choice([-3, 0, 1, 7, 1000, 20010, 20011, 2 ** 31 - 1], rows)
    p = rng.choice([-0.5, 0.0, 0.1, 0.9, 1.0, 1.5], rows)
    m = rng.choice([-1.0, 0.0, 0.01, 0.5, 1.0], rows)
    check_sample(gh, l, t, k, p, m)


@pytest.mark.gpu
def test_sample_nan_settings_filter_nothing(gh):
    rng = np.random.default_rng(22)
    l = rng.standard_normal((3, 5000)).astype(F32)
    a = check_sample(gh, l, u=[0.1, 0.5, 0.9])
    import torch

    tokens = torch.empty(3, dtype=torch.int32, device="cuda")
    nan = cuda(np.full(3, np.nan, F32))
    gh.sample(tokens, None, cuda(l), 0, 3, 5000, gemma_hip.sampling(None, None, nan, nan),
              cuda(np.array([0.1, 0.5, 0.9], F32)), None, stream())
    torch.cuda.synchronize()
    assert np.array_equal(tokens.cpu().numpy(), a)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [300, 5000, 262144])
def test_sample_ties_and_values_that_are_not_finite(gh, vocab):
    rng = np.random.default_rng(23)
    l = np.zeros((12, vocab), F32)
    l[1] = rng.integers(0, 3, vocab)               # few values, many ties
    l[2] = np.where(rng.random(vocab) < 0.5, 0.0, -0.0)
    l[3] = -np.inf                                 # nothing
    l[4] = np.nan
    l[5] = -np.inf
    l[5, vocab - 2] = -3e38                        # one only
    l[6] = rng.standard_normal(vocab)
    l[6, ::7] = np.nan
    l[7] = rng.standard_normal(vocab)
    l[7, ::11] = -np.inf
    l[8] = rng.standard_normal(vocab)
    l[8, [5, 17, vocab - 1]] = np.inf              # infinities take all
    l[9] = np.where(np.arange(vocab) % 2, 3.4e38, -3.4e38)
    l[10] = 1e-40 * rng.integers(-3, 4, vocab)     # subnormal ones
    l[11] = np.nextafter(F32(5.0), F32(9.0))
    l[11, vocab // 2] = 5.0
    for k, p, u in ((None, None, 0.6), (7, None, 0.9), (None, 0.3, 0.99), (vocab // 3, 0.7, 0.5),
                    (None, None, 0.0)):
        check_sample(gh, l, 1.0, k, p, None, u=np.full(12, u, F32))


@pytest.mark.gpu
def test_sample_follows_the_distribution(gh):
    """Tokens over a grid of random numbers: each as often as its share says."""
    n = 4096
    l = np.log(np.array([0.5, 0.1, 0.25, 0.15])).astype(F32)
    u = ((np.arange(n) + 0.5) / n).astype(F32)
    got = check_sample(gh, np.tile(l, (n, 1)), u=u)
    assert np.abs(np.bincount(got, minlength=4) / n - np.exp(l)).max() <= 2 / n


# ---- streams, graphs, threads, workspaces ---------------------------------------


@pytest.mark.gpu
def test_workspaces_are_checked(gh):
    import torch

    rng = np.random.default_rng(31)
    p = Paged([(1, 9000)], 1, 256, 64, CACHE_I8, rng)
    p.fill(rng)
    c = p.device()
    need = gh.cache_attention_work(c, p.batch(), 4, 0, 0)
    q = torch.randn((1, 1024), device="cuda")
    out = torch.empty_like(q)
    if need:
        for work in (torch.empty(need - 1, dtype=torch.uint8, device="cuda"),
                     torch.empty(need + 16, dtype=torch.uint8, device="cuda")[16:]):
            with pytest.raises(gemma_hip.GemmaHipError, match="workspace"):
                gh.cache_attention(out, q, 0, c, p.batch(), 4, 0, 0.1, 0.0, False, 0, work,
                                   stream())
    need = gh.sample_work(2, 262144)
    if need:
        l = torch.randn((2, 262144), device="cuda")
        tok = torch.empty(2, dtype=torch.int32, device="cuda")
        u = torch.rand(2, device="cuda")
        with pytest.raises(gemma_hip.GemmaHipError, match="workspace"):
            gh.sample(tok, None, l, 0, 2, 262144, None, u,
                      torch.empty(need - 1, dtype=torch.uint8, device="cuda"), stream())


@pytest.mark.gpu
def test_workspace_contents_do_not_matter(gh):
    """A workspace filled with NaN bits gives the bits of one filled with zeros, and
    two runs give the same."""
    import torch

    rng = np.random.default_rng(32)
    p = Paged([(1, 3000), (1, 40), (60, 700)], 1, 256, 64, CACHE_I8, rng)
    p.fill(rng)
    c = p.device()
    q = torch.randn((p.rows, 1024), device="cuda")
    l = torch.randn((3, 100003), device="cuda")
    u = torch.rand(3, device="cuda")
    got = []
    for fill in (0, 255, 127, 255):
        out = torch.empty((p.rows, 1024), device="cuda")
        tok = torch.empty(3, dtype=torch.int32, device="cuda")
        prob = torch.empty(3, device="cuda")
        w = [torch.full((max(1, n),), fill, dtype=torch.uint8, device="cuda")
             for n in (gh.cache_attention_work(c, p.batch(), 4, 0, 0), gh.sample_work(3, 100003))]
        gh.cache_attention(out, q, 0, c, p.batch(), 4, 0, 0.06, 0.0, False, 0, w[0], stream())
        gh.sample(tok, prob, l, 0, 3, 100003, None, u, w[1], stream())
        torch.cuda.synchronize()
        got.append((out, tok, prob))
    for g in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got[0], g))


@pytest.mark.gpu
def test_capture_without_a_workspace_is_refused(gh):
    import torch

    rng = np.random.default_rng(33)
    p = Paged([(1, 9000)], 1, 256, 64, CACHE_I8, rng)
    p.fill(rng)
    c = p.device()
    q, out = torch.randn((1, 1024), device="cuda"), torch.empty((1, 1024), device="cuda")
    if gh.cache_attention_work(c, p.batch(), 4, 0, 0) == 0:
        pytest.skip("no workspace at this size")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        q2 = q + 1.0
        with pytest.raises(gemma_hip.GemmaHipError, match="captured"):
            gh.cache_attention(out, q2, 0, c, p.batch(), 4, 0, 0.1, 0.0, False, 0, None, stream())
    graph.replay()
    torch.cuda.synchronize()


class Model:
    """A toy of one layer: tables give each token's q, k, v; logits are the attention's
    output times a matrix.  Run by the library, and in numpy."""

    heads, kv, hd, vocab = 4, 1, 128, 1000

    def __init__(self, rng):
        def t(*s):
            return rng.standard_normal(s).astype(F32)

        self.q, self.k, self.v = (t(self.vocab, n * self.hd) for n in (self.heads, self.kv, self.kv))
        self.w = (t(self.vocab, self.heads * self.hd) * 0.3).astype(F32)


@pytest.mark.gpu
@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("kind", sorted(KINDS))
def test_a_served_batch(gh, kind, graph):
    """Prompts of three sequences behind a shared prefix, then 12 sampled tokens of
    each: write, attend, project, sample, with lengths and tokens kept on the GPU,
    eagerly or as one graph replayed.  Against the same in numpy, 64 bits from the
    codes on."""
    import torch

    kind, rng = KINDS[kind], np.random.default_rng(41)
    m = Model(rng)
    heads, kv, hd, vocab, page, shared, steps = m.heads, m.kv, m.hd, m.vocab, 16, 32, 12
    asc = hd ** -0.5
    prompts = [rng.integers(0, vocab, n) for n in (35, 51, 40)]
    for x in prompts[1:]:
        x[:shared] = prompts[0][:shared]
    B = len(prompts)
    width = 5
    table = np.zeros((B, width), np.int32)
    ids = rng.permutation(40).astype(np.int32)
    for b in range(B):
        table[b] = np.concatenate([ids[:2], ids[2 + 3 * b:5 + 3 * b]])
    u = rng.random((steps + 1, B)).astype(F32)
    temp, top_k, top_p, min_p = ([0.9, 1.2, 0.0], [0, 50, 0], [0.9, 1.0, 1.0], [0.0, 0.02, 0.0])

    # the library
    kc, vc = (torch.full((40, kv, page, hd), 0x7f, dtype=torch.uint8, device="cuda") for _ in "kv")
    ks, vs = (torch.full((40, kv, page), float("nan"), device="cuda") for _ in "kv")
    cache = gemma_hip.cache(kc, vc, ks, vs, kind, 40, page, kv, hd)
    tab, tq, tk, tv, w = (cuda(a) for a in (table, m.q, m.k, m.v, m.w))
    settings = gemma_hip.sampling(cuda(np.array(temp, F32)), cuda(np.array(top_k, np.int32)),
                                  cuda(np.array(top_p, F32)), cuda(np.array(min_p, F32)))
    s = torch.cuda.Stream()
    got = []
    with torch.cuda.stream(s):
        n = [len(x) for x in prompts]
        ln = cuda(np.array(n, np.int32))
        row0 = cuda(np.concatenate([[0], np.cumsum(n)]).astype(np.int32))
        tok = cuda(np.concatenate(prompts))
        total = sum(n)
        # the first sequence brings the prefix, then all bring the rest: here the
        # shared pages get the same codes from each, one sequence at a time
        for b in range(B):
            one = gemma_hip.batch(tab[b:b + 1], ln[b:b + 1], cuda(np.array([0, n[b]], np.int32)),
                                  1, width, n[b], n[b], n[b])
            t = cuda(prompts[b])
            gh.cache_write(cache, one, tk[t], 0, tv[t], 0, s.cuda_stream)
        rows = torch.empty((total, heads * hd), device="cuda")
        batch = gemma_hip.batch(tab, ln, row0, B, width, total, max(n), max(n))
        gh.cache_attention(rows, tq[tok], 0, cache, batch, heads, 0, asc, 0.0, False, shared, None,
                           s.cuda_stream)
        last = rows[(row0[1:] - 1).long()].contiguous()
        logits = torch.empty((B, vocab), device="cuda")
        tokens = torch.empty(B, dtype=torch.int32, device="cuda")
        du = cuda(u)
        gh.matmul_f32(logits, 0, w, 0, last, 0, B, vocab, heads * hd, s.cuda_stream)
        gh.sample(tokens, None, logits, 0, B, vocab, settings, du[0], None, s.cuda_stream)
        got.append(tokens.cpu().numpy().copy())
        # single tokens
        row1 = cuda(np.arange(B + 1, dtype=np.int32))
        batch = gemma_hip.batch(tab, ln, row1, B, width, B, 1, width * page)
        q, k, v = (torch.empty((B, x * hd), device="cuda") for x in (heads, kv, kv))
        o = torch.empty((B, heads * hd), device="cuda")
        cur = torch.empty(B, device="cuda")
        wa, ws = (torch.empty(max(1, x), dtype=torch.uint8, device="cuda") for x in
                  (gh.cache_attention_work(cache, batch, heads, 0, shared),
                   gh.sample_work(B, vocab)))

        def step():
            st = torch.cuda.current_stream().cuda_stream
            t = tokens.long()
            q.copy_(tq[t])
            k.copy_(tk[t])
            v.copy_(tv[t])
            ln.add_(1)
            gh.cache_write(cache, batch, k, 0, v, 0, st)
            gh.cache_attention(o, q, 0, cache, batch, heads, 0, asc, 0.0, False, shared, wa, st)
            gh.matmul_f32(logits, 0, w, 0, o, 0, B, vocab, heads * hd, st)
            gh.sample(tokens, None, logits, 0, B, vocab, settings, cur, ws, st)

    if graph:
        s.synchronize()
        keep = tokens.clone(), ln.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            step()
        tokens.copy_(keep[0])
        ln.copy_(keep[1])
        torch.cuda.synchronize()
    for i in range(steps):
        with torch.cuda.stream(s):
            cur.copy_(du[i + 1])
            g.replay() if graph else step()
            got.append(tokens.cpu().numpy().copy())

    # numpy
    seqs, close = [list(x) for x in prompts], 0
    for i in range(steps + 1):
        for b in range(B):
            x = np.array(seqs[b])
            kk, vv = (values(*quantise(a[x], kind), kind) for a in (m.k, m.v))
            at = np.concatenate([attend(m.q[x[-1], h * hd:(h + 1) * hd], kk, vv, len(x) - 1,
                                        len(x), 0, asc, 0.0, False)[0] for h in range(heads)])
            tok, _, margin = draw_token((m.w.astype(F64) @ at).astype(F32), F64(F32(temp[b])),
                                        top_k[b], F64(F32(top_p[b])), F64(F32(min_p[b])),
                                        F64(u[i, b]))
            # the logits are within about 1e-5: a draw nearer than that to one of some
            # thousand borders may fall on the other side (2% of them are)
            close += margin <= 1e-5
            assert got[i][b] == tok or margin <= 1e-5, (i, b, margin)
            seqs[b].append(int(got[i][b]))
    assert close <= 4


@pytest.mark.gpu
def test_graph_replays_follow_the_tables(gh):
    """One captured attention call, replayed for other lengths, pages and rows, with
    eager work between: each replay is the eager call's bits."""
    import torch

    rng = np.random.default_rng(42)
    p = Paged([(1, 900)] * 3, 1, 256, 16, CACHE_I8, rng)
    p.fill(rng)
    c = p.device()
    batch = p.batch()
    q = torch.randn((3, 1024), device="cuda")
    out, eager = torch.empty((3, 1024), device="cuda"), torch.empty((3, 1024), device="cuda")
    work = torch.empty(max(1, gh.cache_attention_work(c, batch, 4, 0, 0)), dtype=torch.uint8,
                       device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        gh.cache_attention(out, q, 0, c, batch, 4, 0, 0.06, 0.0, False, 0, work, stream())
    for lens in ([900, 500, 40], [1, 0, 899], [33, 32, 31], [900, 500, 40], [16, 17, 500]):
        p.dlen.copy_(cuda(np.array(lens, np.int32)))
        if lens[0] == 33:
            p.tab.copy_(cuda(p.table[[1, 0, 2]]))
        q.normal_()
        g.replay()
        gh.cache_attention(eager, q, 0, c, batch, 4, 0, 0.06, 0.0, False, 0, None, stream())
        torch.cuda.synchronize()
        assert torch.equal(out, eager), lens
        assert (out[1] == 0).all() == (lens[1] == 0)


@pytest.mark.gpu
def test_two_streams_and_threads(gh):
    """Calls from four threads, each on a stream of its own, without workspaces of
    their own: each thread's results are its own."""
    import torch

    rng = np.random.default_rng(43)
    p = Paged([(1, 4000), (1, 700), (20, 300)], 1, 256, 64, CACHE_I8, rng)
    p.fill(rng)
    c, batch = p.device(), p.batch()
    qs = [torch.randn((p.rows, 1024), device="cuda") for _ in range(4)]
    ls = [torch.randn((3, 50000), device="cuda") for _ in range(4)]
    us = [torch.rand(3, device="cuda") for _ in range(4)]

    def both(i, st):
        out = torch.empty((p.rows, 1024), device="cuda")
        tok = torch.empty(3, dtype=torch.int32, device="cuda")
        gh.cache_attention(out, qs[i], 0, c, batch, 4, 0, 0.06, 0.0, False, 0, None, st)
        gh.sample(tok, None, ls[i], 0, 3, 50000, None, us[i], None, st)
        return out, tok

    want = [both(i, stream()) for i in range(4)]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(10):
                got = both(i, s.cuda_stream)
                s.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    bad.append(i)

    ts = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not bad


@pytest.mark.gpu
def test_offsets_pass_32_bits(gh):
    """A cache of more than 4 GiB of codes and 2^32 values, the sequence in its last
    pages."""
    import torch

    kind, hd, kv, page = CACHE_I8, 256, 4, 256
    npages = (1 << 32) // (kv * page * hd) + 3
    codes = [torch.zeros((npages, kv, page, hd), dtype=torch.uint8, device="cuda") for _ in "kv"]
    scales = [torch.zeros((npages, kv, page), device="cuda") for _ in "kv"]
    c = gemma_hip.cache(*codes, *scales, kind, npages, page, kv, hd)
    n = 300
    table = cuda(np.array([[npages - 1, npages - 2]], np.int32))
    ln, row0 = cuda(np.array([n], np.int32)), cuda(np.array([0, n], np.int32))
    b = gemma_hip.batch(table, ln, row0, 1, 2, n, n, n)
    k, v = (torch.randn((n, kv * hd), device="cuda") for _ in "kv")
    gh.cache_write(c, b, k, 0, v, 0, stream())
    rk, rv = torch.empty_like(k), torch.empty_like(v)
    gh.cache_read(c, b, rk, 0, rv, 0, stream())
    q = torch.randn((n, 8 * hd), device="cuda")
    out = torch.empty_like(q)
    gh.cache_attention(out, q, 0, c, b, 8, 0, 0.0625, 0.0, False, 0, None, stream())
    torch.cuda.synchronize()
    kk, vv = (values(*quantise(x.cpu().numpy().reshape(n, kv, hd), kind), kind) for x in (k, v))
    assert np.array_equal(rk.cpu().numpy().reshape(n, kv, hd), kk)
    assert np.array_equal(rv.cpu().numpy().reshape(n, kv, hd), vv)
    qn, got = q.cpu().numpy(), out.cpu().numpy()
    for i in (0, 100, n - 1):
        for h in range(8):
            want, vmax = attend(qn[i, h * hd:(h + 1) * hd], kk[:, h // 2], vv[:, h // 2], i, n, 0,
                                0.0625, 0.0, False)
            assert np.abs(got[i, h * hd:(h + 1) * hd] - want).max() <= ATT_TOL * vmax
    del codes, scales


@pytest.mark.gpu
def test_timed_as_the_reference_ops(gh):
    import torch

    rng = np.random.default_rng(44)
    p = Paged([(2, 40)], 1, 128, 16, CACHE_I8, rng)
    p.fill(rng)
    c = p.device()
    x = torch.randn((2, 128), device="cuda")
    o = torch.empty((2, 128), device="cuda")
    tok = torch.empty(1, dtype=torch.int32, device="cuda")
    gh.perf_enable(True)
    try:
        gh.perf_phase("decode")
        gh.cache_write(c, p.batch(), x, 0, x, 0, stream())
        gh.cache_attention(o, x, 0, c, p.batch(), 1, 0, 0.1, 0.0, False, 0, None, stream())
        gh.sample(tok, None, torch.randn((1, 500), device="cuda"), 0, 1, 500, None,
                  torch.rand(1, device="cuda"), None, stream())
        perf = gh.perf_read()["decode"]
    finally:
        gh.perf_enable(False)
    assert {n: perf[n][1] for n in ("quantize_act", "softmax", "sample_from_logits")} == \
        {"quantize_act": 1, "softmax": 1, "sample_from_logits": 1}
