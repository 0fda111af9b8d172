"""Batches over a paged key/value cache for the tests: made on the host, run through the C ABI, and
computed in 64 bits from the definition."""
import ctypes

import numpy as np

import cachepotato_amd as C

F32, F16, BF16 = C.T_F32, C.T_F16, C.T_BF16
NAMES = {F32: "f32", F16: "f16", BF16: "bf16"}
# the largest relative error of one rounding to the type
HALF_STEP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}


def to_type(x, t):
    """float array -> the array of the type's bits (round to nearest even)"""
    x = np.asarray(x, np.float32)
    if t == F32:
        return x
    if t == F16:
        return x.astype(np.float16)
    u = np.ascontiguousarray(x).view(np.uint32).astype(np.uint64)
    nan = np.isnan(x)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(nan, np.uint16(0x7FC0), r)


def values(a, t):
    """the values that an array of the type's bits stands for, float64"""
    if t == BF16:
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


def storage(t):
    return {F32: np.float32, F16: np.float16, BF16: np.uint16}[t]


class Batch:
    """Sequences (len, new) over a pool whose every slot starts as NaN. The pool's order is (page,
    slot, head) or (page, head, slot), with `gap` unused elements behind each of its rows."""

    def __init__(self, seqs, KV, HD, page, ctype, by_head=False, gap=0, T=None, first_row=0, seed=0,
                 max_pages=None, spare=2):
        self.rng = np.random.default_rng(seed)
        self.seqs, self.KV, self.HD, self.page, self.ctype = seqs, KV, HD, page, ctype
        self.S = len(seqs)
        self.off = np.cumsum([first_row] + [n for _, n in seqs]).astype(np.int32)
        self.len = np.array([L for L, _ in seqs], np.int32)
        self.T = int(self.off[-1]) if T is None else T
        need = [-(-L // page) for L, _ in seqs]
        self.max_pages = max(need + [1]) if max_pages is None else max_pages
        self.n_pages = sum(need) + spare
        ids = self.rng.permutation(self.n_pages).astype(np.int32)
        # entries that no sequence has are no page ids at all
        self.pages = np.full((self.S, self.max_pages), -7, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.pages[s, :n] = ids[at:at + n]
            at += n
        self.slot_stride, self.head_stride = (HD + gap, page * (HD + gap)) if by_head else (KV * HD + gap, HD)
        self.page_stride = KV * page * (HD + gap) if by_head else page * (KV * HD + gap)
        n = self.n_pages * self.page_stride
        self.k = to_type(np.full(n, np.nan), ctype)
        self.v = self.k.copy()
        self.dev = {}

    def where(self, s, j):
        """the elements of head 0 .. KV-1 of token j of sequence s: (KV, HD) indices"""
        base = int(self.pages[s, j // self.page]) * self.page_stride + j % self.page * self.slot_stride
        return base + np.arange(self.KV)[:, None] * self.head_stride + np.arange(self.HD)

    def fill(self, sigma=1.0):
        """every token that a sequence holds: normal keys and values"""
        for s, (L, _) in enumerate(self.seqs):
            for j in range(L):
                w = self.where(s, j)
                self.k[w] = to_type(self.rng.standard_normal(w.shape) * sigma, self.ctype)
                self.v[w] = to_type(self.rng.standard_normal(w.shape) * 0.9, self.ctype)
        return self

    def held(self, s, which):
        """(len, KV, HD) values of a sequence's keys or values"""
        a = self.k if which == "k" else self.v
        L = self.seqs[s][0]
        out = np.empty((L, self.KV, self.HD))
        for j in range(L):
            out[j] = values(a[self.where(s, j)], self.ctype)
        return out

    # ---- device side

    def upload(self):
        for name in ("k", "v", "pages", "off", "len"):
            if name in self.dev:
                self.dev[name].upload(getattr(self, name))
            else:
                self.dev[name] = C.to_device(getattr(self, name))
        return self

    def cache(self):
        return C.PagedCache(self.KV, self.HD, self.ctype, self.page, self.n_pages, self.page_stride,
                            self.slot_stride, self.head_stride, self.dev["k"].ptr, self.dev["v"].ptr)

    def batch(self, max_new=None):
        n = max([n for _, n in self.seqs] + [0]) if max_new is None else max_new
        return C.PagedBatch(self.S, self.T, n, self.max_pages, self.dev["pages"].ptr, self.dev["off"].ptr,
                            self.dev["len"].ptr)

    def pool(self):
        """the pool as the device has it now"""
        dt = storage(self.ctype)
        return tuple(self.dev[x].download(dt, self.k.size) for x in ("k", "v"))

    def close(self):
        for b in self.dev.values():
            b.close()
        self.dev = {}


class Workspace:
    def __init__(self, H, KV, HD):
        self.ptr = C.lib().cpg_paged_ws_create(H, KV, HD)
        if not self.ptr:
            raise C.CPGError(C.last_error())

    def status(self):
        return C.lib().cpg_paged_ws_status(self.ptr)

    def close(self):
        C.lib().cpg_paged_ws_destroy(self.ptr)


def attend(b, ws, q, H, type_, window=0, scale=0.0, ld=None, ldo=None, max_new=None, lse=True):
    """q (T, H, HD) values -> (out (T, H, HD) as the type's bits, lse (T, H)); rows that nothing
    writes keep their NaN"""
    T, HD = b.T, b.HD
    ld, ldo = ld or H * HD, ldo or H * HD
    qh = np.zeros((max(T, 1), ld), storage(type_))
    qh[:T, :H * HD] = to_type(q.reshape(T, H * HD), type_)
    oh = to_type(np.full((max(T, 1), ldo), np.nan), type_)
    dq, do, dl = C.to_device(qh), C.to_device(oh), C.to_device(np.full((max(T, 1), H), np.nan, np.float32))
    rc = C.lib().cpg_paged_attn(ctypes.byref(b.cache()), ctypes.byref(b.batch(max_new)), type_, H, dq.ptr, ld,
                                scale, window, do.ptr, ldo, dl.ptr if lse else None, ws.ptr)
    C.check(rc, "cpg_paged_attn")
    C.sync()
    out = do.download(storage(type_), max(T, 1) * ldo).reshape(-1, ldo)[:T, :H * HD].reshape(T, H, HD)
    got = dl.download(np.float32, max(T, 1) * H).reshape(-1, H)[:T]
    for d in (dq, do, dl):
        d.close()
    return out, got


def attention64(b, q, H, window=0, scale=0.0):
    """(out, lse, and of each row the largest |v| and the sum |q||k| scale that it can meet): the
    definition in 64 bits; NaN for rows of no sequence"""
    T, HD, G = b.T, b.HD, H // b.KV
    scale = scale or HD ** -0.5
    out, lse = np.full((T, H, HD), np.nan), np.full((T, H), np.nan)
    vmax, smax = np.zeros((T, H)), np.zeros((T, H))
    for s, (L, n) in enumerate(b.seqs):
        k, v = b.held(s, "k"), b.held(s, "v")
        for i in range(n):
            t, p = int(b.off[s]) + i, L - n + i
            lo = max(0, p - window + 1) if window else 0
            if p < 0:
                out[t], lse[t] = 0.0, -np.inf
                continue
            for h in range(H):
                kk, vv = k[lo:p + 1, h // G], v[lo:p + 1, h // G]
                x = kk @ q[t, h] * scale
                m = x.max()
                e = np.exp(x - m)
                out[t, h] = e @ vv / e.sum()
                lse[t, h] = m + np.log(e.sum())
                vmax[t, h] = np.abs(vv).max()
                smax[t, h] = np.sqrt((kk * kk).sum(1).max() * (q[t, h] @ q[t, h])) * scale
    return out, lse, vmax, smax
