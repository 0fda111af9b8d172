"""cpg_paged_append and cpg_paged_attn on the GPU, against the definition in 64 bits.

Tolerances. A score is a sum of HD products in fp32: its rounding errors add up like a random walk,
so e_s = 2^-24 sqrt(HD) |q||k| scale + 2^-22 |q||k| scale / sqrt(HD), the second term for f32
queries in 22-bit pieces. A weight then is off by e_s (its own score) + e_s (the maximum's) + 2^-22
(the power of two), relatively, and the sums over n keys by 2^-24 sqrt(n) more, twice. Times the
largest |v| this bounds an output; 16-bit outputs add half a step for the weights and half a step for
the output, of |v| at most. f32 caches of more than 16 rows per kv head hold keys, values and weights
in 22-bit pieces: 2^-22 |v| more. lse: e_s + 2^-22 of its size and of 1."""
import ctypes

import numpy as np
import pytest

import cachepotato_amd as C
from tests.paged_helpers import (BF16, F16, F32, HALF_STEP, NAMES, Batch, Workspace, attend, attention64,
                                 storage, to_type, values)

pytestmark = pytest.mark.gpu

COMBOS = [(F32, F32), (F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)]


@pytest.fixture(autouse=True, params=[C.PAGED_AUTO, C.PAGED_FEW, C.PAGED_MANY], ids=["auto", "few", "many"])
def mode(request):
    """every test with the kernel that the batch chooses, and with each of the two"""
    if request.param != C.PAGED_AUTO and "append" in request.node.name:
        pytest.skip("no attention")
    C.check(C.lib().cpg_paged_attn_mode(request.param))
    yield request.param
    C.check(C.lib().cpg_paged_attn_mode(C.PAGED_AUTO))


def say(*a):
    print(*a, flush=True)


def bounds(type_, HD, n, vmax, smax):
    es = 2.0 ** -24 * np.sqrt(HD) * smax + 2.0 ** -22 * smax / np.sqrt(HD)
    rel = 2 * es + 2.0 ** -22 + 2 * 2.0 ** -24 * np.sqrt(n) + 2.0 ** -22
    if type_ != F32:
        rel = rel + 2 * HALF_STEP[type_]
    return (rel * vmax)[:, :, None], es


def queries(b, H, type_, seed=5, sigma=1.0):
    q = np.random.default_rng(seed).standard_normal((b.T, H, b.HD)) * sigma
    return values(to_type(q, type_), type_)


def compare(b, q, H, type_, got, lse, window=0, scale=0.0, rows=None):
    want, wlse, vmax, smax = attention64(b, q, H, window, scale)
    n = max([L for L, _ in b.seqs] + [1])
    tol, es = bounds(type_, b.HD, n, vmax, smax)
    g = values(got, type_)
    rows = np.arange(b.T) if rows is None else rows
    assert np.array_equal(np.isnan(g[rows]), np.isnan(want[rows]))
    own = rows[~np.isnan(want[rows]).any((1, 2))]
    err = np.abs(g[own] - want[own])
    worst = float((err / np.maximum(tol[own], 1e-300)).max()) if own.size else 0.0
    say(f"   {NAMES[type_]}/{NAMES[b.ctype]} HD={b.HD} H={H} KV={b.KV} page={b.page} window={window}: "
        f"max err {err.max() if own.size else 0:.2e}, {worst:.2f} of the bound")
    assert (err <= tol[own]).all()
    if lse is not None:
        fin = np.isfinite(wlse[own])
        assert np.array_equal(fin, np.isfinite(lse[own]))
        assert (lse[own][~fin] == -np.inf).all()
        le = np.abs(lse[own][fin] - wlse[own][fin])
        assert (le <= es[own][fin] + 2.0 ** -22 * (1 + np.abs(wlse[own][fin]))).all()


def run(seqs, H, KV, HD, page, type_, ctype, window=0, scale=0.0, max_new=None, sigma=1.0, **kw):
    say(f"case seqs={seqs} H={H} KV={KV} HD={HD} page={page} {NAMES[type_]}/{NAMES[ctype]} window={window} {kw}")
    b = Batch(seqs, KV, HD, page, ctype, **kw).fill(sigma).upload()
    ws = Workspace(H, KV, HD)
    try:
        q = queries(b, H, type_)
        out, lse = attend(b, ws, q, H, type_, window, scale, max_new=max_new)
        assert ws.status() == 0
        compare(b, q, H, type_, out, lse, window, scale)
        return out
    finally:
        ws.close()
        b.close()


# ---------------------------------------------------------------- attention

DECODE = [(1, 1), (2, 1), (15, 1), (16, 1), (17, 1), (127, 1), (128, 1), (129, 1), (300, 1)]
CHUNKS = [(1, 1), (5, 5), (40, 33), (129, 2), (200, 70), (131, 131)]


@pytest.mark.parametrize("type_,ctype", COMBOS)
@pytest.mark.parametrize("HD", [64, 96, 128, 192, 256])
def test_decode_lengths(cpg, type_, ctype, HD):
    run(DECODE, 8, 2, HD, 16, type_, ctype)


@pytest.mark.parametrize("type_,ctype", COMBOS)
@pytest.mark.parametrize("HD", [64, 96, 128, 192, 256])
def test_chunks(cpg, type_, ctype, HD):
    run(CHUNKS, 4, 2, HD, 16, type_, ctype, by_head=HD == 128, gap=8)


@pytest.mark.parametrize("H,KV", [(1, 1), (3, 3), (6, 2), (5, 1), (8, 1), (12, 1), (16, 1), (21, 1), (40, 2),
                                  (150, 1), (32, 4)])
@pytest.mark.parametrize("type_,ctype", [(F32, F32), (BF16, BF16)])
def test_head_layouts(cpg, H, KV, type_, ctype):
    run([(70, 1), (33, 3), (140, 20)], H, KV, 64, 8, type_, ctype)


@pytest.mark.parametrize("page", [1, 2, 4, 8, 16, 64, 1024])
@pytest.mark.parametrize("type_,ctype", [(F32, F32), (F32, F16), (BF16, BF16)])
def test_pages(cpg, page, type_, ctype):
    run([(1, 1), (37, 1), (100, 40), (259, 9)], 8, 2, 128, page, type_, ctype, by_head=page == 8)


@pytest.mark.parametrize("window", [1, 2, 7, 64, 100, 128, 5000, 2 ** 31 - 1])
@pytest.mark.parametrize("type_,ctype", [(F32, F32), (F32, BF16), (F16, F16)])
def test_window(cpg, window, type_, ctype):
    run([(300, 1), (90, 90), (260, 30), (3, 3)], 4, 2, 64, 16, type_, ctype, window=window)


@pytest.mark.parametrize("window", [1, 5, 40])
def test_window_and_rows_without_keys(cpg, window):
    """sequences shorter than their new rows, under a window"""
    run([(3, 9), (40, 70), (0, 2), (50, 50), (60, 1)], 8, 2, 64, 16, F32, F32, window=window)
    run([(3, 9), (40, 70), (0, 2), (50, 50), (60, 1)], 4, 2, 64, 16, BF16, BF16, window=window)


def test_rows_that_do_not_ascend(cpg):
    """offsets that give the same rows to many sequences, whose units would pass every bound: nothing
    is written, with one sequence, within a wavefront's reach and beyond"""
    for S in (2, 64, 300):
        b = Batch([(60, 4)] * S, 1, 64, 16, F32).fill().upload()
        b.off = np.array([0, b.T] * S, np.int32)[:S + 1]
        b.upload()
        ws = Workspace(4, 1, 64)
        out, lse = attend(b, ws, np.zeros((b.T, 4, 64)), 4, F32)
        assert ws.status() == 1 and np.isnan(out).all() and np.isnan(lse).all()
        ws.close()
        b.close()


def test_window_pages_are_not_looked_at(cpg):
    """pages behind every row's window may have been given to others: their ids may be anything"""
    b = Batch([(400, 1), (390, 21)], 2, 64, 16, F32).fill()
    want_held = b.pages.copy()
    q = queries(b, 4, F32)
    want = attention64(b, q, 4, 50)
    for s, (L, n) in enumerate(b.seqs):
        b.pages[s, :(L - n - 50 + 1) // 16] = [-1, 1 << 30][s]
    b.upload()
    ws = Workspace(4, 2, 64)
    out, lse = attend(b, ws, q, 4, F32, 50)
    assert ws.status() == 0
    b.pages = want_held
    compare(b, q, 4, F32, out, lse, 50)
    ws.close()
    b.close()


@pytest.mark.parametrize("type_,ctype", COMBOS)
def test_no_rows_and_rows_without_keys(cpg, type_, ctype):
    """sequences without new tokens, of no tokens at all, and shorter than their new rows"""
    run([(9, 0), (0, 3), (5, 8), (40, 0), (2, 70), (30, 1), (0, 0)], 8, 2, 64, 16, type_, ctype)


def test_rows_of_no_sequence_stay(cpg):
    """rows before the first and behind the last sequence keep what they hold (NaN here)"""
    for type_, ctype in COMBOS:
        run([(30, 2), (50, 1), (7, 0)], 8, 2, 128, 16, type_, ctype, T=9, first_row=2)


def test_nothing_to_do(cpg):
    b = Batch([(4, 0)], 2, 64, 16, F32).fill().upload()
    ws = Workspace(4, 2, 64)
    b.T = 0
    attend(b, ws, np.zeros((0, 4, 64)), 4, F32)
    b.T, b.S = 3, 0
    out, _ = attend(b, ws, np.zeros((3, 4, 64)), 4, F32)
    assert np.isnan(out).all()
    b.S = 1                                          # three rows that the one sequence does not have
    out, _ = attend(b, ws, np.zeros((3, 4, 64)), 4, F32)
    assert np.isnan(out).all() and ws.status() == 0
    ws.close()
    b.close()


def test_many_sequences(cpg):
    """more sequences than one round of the scan (256), decode and ragged"""
    rng = np.random.default_rng(3)
    seqs = [(int(rng.integers(1, 60)), 1) for _ in range(700)]
    run(seqs, 4, 1, 64, 8, F32, F16)
    seqs = [(int(n + rng.integers(0, 40)), int(n)) for n in rng.integers(0, 5, 300)]
    run(seqs, 4, 1, 64, 8, BF16, BF16)


@pytest.mark.parametrize("max_new", [0, 1, 1000])
@pytest.mark.parametrize("type_,ctype", COMBOS)
def test_max_new_is_a_hint(cpg, max_new, type_, ctype):
    run([(150, 1), (90, 40), (64, 64)], 8, 1, 128, 16, type_, ctype, max_new=max_new)


@pytest.mark.parametrize("type_,ctype", COMBOS)
def test_scale_and_sizes_of_scores(cpg, type_, ctype):
    """scores up to several hundred (a softmax that is nearly one key's), a scale of one's own"""
    run([(200, 1), (150, 20)], 8, 2, 64, 16, type_, ctype, scale=0.7, sigma=3.0)
    run([(200, 1), (150, 20)], 8, 2, 64, 16, type_, ctype, scale=1e-3)


@pytest.mark.parametrize("qs", [1e-12, 1e-4, 1e4, 1e12])
@pytest.mark.parametrize("ctype", [F32, F16, BF16])
def test_query_range(cpg, qs, ctype):
    """f32 queries of any size that the scale brings back: their 16-bit pieces follow the row's size"""
    b = Batch([(100, 1), (80, 40)], 2, 64, 16, ctype).fill().upload()
    ws = Workspace(8, 2, 64)
    q = queries(b, 8, F32) * np.float64(np.float32(qs))
    q = q.astype(np.float32).astype(np.float64)
    out, lse = attend(b, ws, q, 8, F32, scale=0.125 / qs)
    compare(b, q, 8, F32, out, lse, 0, float(np.float32(0.125 / qs)))
    ws.close()
    b.close()


@pytest.mark.parametrize("ks,vs", [(1e-30, 1e-30), (1e-5, 1e-4), (1e5, 1e6), (1e30, 1e30), (1.0, 1e-7), (1.0, 1e7)])
@pytest.mark.parametrize("HD", [64, 128, 192])
def test_cache_range(cpg, HD, ks, vs):
    """f32 caches take any size of keys and values; the scores are of order one throughout"""
    for seqs in ([(150, 1), (90, 60), (200, 33)], [(700, 40)]):
        b = Batch(seqs, 2, HD, 16, F32).fill()
        b.k *= np.float32(ks)
        b.v *= np.float32(vs)
        b.upload()
        ws = Workspace(8, 2, HD)
        q = queries(b, 8, F32, sigma=1 / ks)
        out, lse = attend(b, ws, q, 8, F32)
        assert ws.status() == 0
        compare(b, q, 8, F32, out, lse)
        ws.close()
        b.close()


@pytest.mark.parametrize("window", [0, 90])
def test_cache_range_over_a_sequence(cpg, window):
    """values that grow and fall over 2^40, keys over 2^8, from token to token, some of them zero"""
    b = Batch([(640, 200), (640, 1)], 2, 64, 16, F32).fill()
    for s in range(2):
        for j in range(640):
            w = b.where(s, j)
            b.v[w] *= np.float32(2.0 ** (20 - abs(j - 320) / 8)) if j % 50 > 20 or j > 500 else np.float32(0)
            b.k[w] *= np.float32(2.0 ** (j % 9 - 4))
    b.upload()
    ws = Workspace(4, 2, 64)
    q = queries(b, 4, F32, sigma=0.1)
    out, lse = attend(b, ws, q, 4, F32, window)
    compare(b, q, 4, F32, out, lse, window)
    ws.close()
    b.close()


@pytest.mark.parametrize("type_,ctype", COMBOS)
@pytest.mark.parametrize("window", [0, 30])
def test_what_a_row_does_not_see_does_not_reach_it(cpg, type_, ctype, window):
    """infinities and NaN in later tokens' keys and values (and, with a window, in earlier ones'):
    rows that see them become NaN or infinite, the others keep their bits"""
    seqs = [(60, 1), (75, 40), (140, 9)]
    b = Batch(seqs, 2, 64, 16, ctype).fill().upload()
    ws = Workspace(8, 2, 64)
    q = queries(b, 8, type_)
    clean, clean_lse = attend(b, ws, q, 8, type_, window)
    bad = {1: 60, 2: 137}                            # token of the sequence; rows at p >= see it
    for s, j in bad.items():
        w = b.where(s, j)
        x = to_type(np.array([np.nan, np.inf, -np.inf]), ctype)
        b.v[w[:, 5]], b.v[w[:, 6]], b.v[w[:, 7]] = x
        b.k[w[:, 3]] = x[s % 2]
    b.upload()
    out, lse = attend(b, ws, q, 8, type_, window)
    for s, (L, n) in enumerate(seqs):
        for i in range(n):
            t, p = int(b.off[s]) + i, L - n + i
            sees = s in bad and p >= bad[s] and (not window or p - window < bad[s])
            if sees:
                assert not np.isfinite(values(out[t], type_)).all(), (s, i)
            else:
                assert np.array_equal(out[t].view(np.uint8), clean[t].view(np.uint8)), (s, i)
                assert np.array_equal(lse[t], clean_lse[t])
    ws.close()
    b.close()


def test_values_alone_wild(cpg):
    """an infinite value among finite keys: the rows that see it have exactly that element infinite"""
    for type_, ctype in COMBOS:
        b = Batch([(50, 30)], 1, 64, 16, ctype).fill()
        b.v[b.where(0, 35)[0, 11]] = to_type(np.array([np.inf]), ctype)[0]
        b.upload()
        ws = Workspace(4, 1, 64)
        out, _ = attend(b, ws, queries(b, 4, type_), 4, type_)
        o = values(out, type_)
        for i in range(30):
            inf = np.zeros((4, 64), bool)
            inf[:, 11] = 20 + i >= 35
            # f32 caches in 16-bit pieces: an infinity's rest is a NaN
            assert np.array_equal(~np.isfinite(o[i]), inf), (NAMES[type_], NAMES[ctype], i)
        ws.close()
        b.close()


def test_long_context_split(cpg):
    """one sequence over many workgroups, and the same batch twice: the same bits"""
    for type_, ctype in ((F32, F32), (F32, BF16), (BF16, BF16)):
        a = run([(5000, 1)], 4, 2, 64, 16, type_, ctype)
        b = run([(5000, 1)], 4, 2, 64, 16, type_, ctype)
        assert np.array_equal(a.view(np.uint8), b.view(np.uint8))
    run([(3000, 10), (20, 1), (1, 1), (900, 300)], 4, 2, 64, 16, F32, F32)


@pytest.mark.parametrize("type_,ctype", [(F32, F32), (BF16, BF16)])
@pytest.mark.parametrize("HD", [64, 96, 128, 192, 256])
def test_item_of_many_pieces(cpg, HD, type_, ctype):
    """an item over all workgroups, its pieces merged in groups, with all of a tile's rows"""
    run([(9000, 1)], 16, 1, HD, 64, type_, ctype)
    run([(7000, 9)], 14, 1, HD, 64, type_, ctype)


def test_strided_rows(cpg):
    """q as the head part of a wider row, out into a wider row"""
    b = Batch([(40, 1), (60, 25)], 2, 128, 16, F32).fill().upload()
    ws = Workspace(8, 2, 128)
    q = queries(b, 8, F32)
    want, wl = attend(b, ws, q, 8, F32)
    got, gl = attend(b, ws, q, 8, F32, ld=12 * 128, ldo=8 * 128 + 4, lse=True)
    assert np.array_equal(want, got) and np.array_equal(wl, gl)
    got, _ = attend(b, ws, q, 8, F32, lse=False)
    assert np.array_equal(want, got)
    ws.close()
    b.close()


@pytest.mark.parametrize("type_,ctype", COMBOS)
def test_bad_page_ids(cpg, type_, ctype):
    """a page id outside the pool: the rows that need it are NaN, the others as they were, and the
    status word says so once"""
    seqs = [(100, 1), (80, 1), (90, 40)]
    b = Batch(seqs, 2, 64, 16, ctype).fill().upload()
    ws = Workspace(8, 2, 64)
    q = queries(b, 8, type_)
    clean, _ = attend(b, ws, q, 8, type_)
    assert ws.status() == 0
    held = b.pages.copy()
    for bad in (-1, b.n_pages, 2 ** 31 - 1, -2 ** 31):
        b.pages = held.copy()
        b.pages[0, 2] = bad                          # tokens 32 .. 47
        b.pages[2, 4] = bad                          # tokens 64 .. 79: rows 14 .. 39 of sequence 2
        b.upload()
        out, lse = attend(b, ws, q, 8, type_)
        o = values(out, type_)
        assert ws.status() == 1 and ws.status() == 0
        assert np.isnan(o[0]).all() and np.isnan(lse[0]).all()
        assert np.array_equal(out[1], clean[1])
        for i in range(40):
            t, p = 2 + i, 50 + i
            if p >= 64:
                assert np.isnan(o[t]).all(), i
            else:
                assert np.array_equal(out[t].view(np.uint8), clean[t].view(np.uint8)), i
    ws.close()
    b.close()


def test_bad_lengths_and_offsets(cpg):
    b = Batch([(20, 1), (30, 20), (40, 1)], 2, 64, 16, F32).fill().upload()
    ws = Workspace(8, 2, 64)
    q = queries(b, 8, F32)
    clean, _ = attend(b, ws, q, 8, F32)
    held = b.len.copy()
    for L in (-1, b.max_pages * 16 + 1, 2 ** 31 - 1, -2 ** 31):
        b.len = held.copy()
        b.len[1] = L
        b.upload()
        out, lse = attend(b, ws, q, 8, F32)
        assert ws.status() == 1
        assert np.isnan(out[1:21]).all() and np.isnan(lse[1:21]).all()
        assert np.array_equal(out[[0, 21]], clean[[0, 21]])
    b.len = held
    off = b.off.copy()
    for change in ((1, -3), (3, 30), (3, 2 ** 31 - 1), (2, -2 ** 31)):
        b.off = off.copy()
        b.off[change[0]] = change[1]
        b.upload()
        attend(b, ws, q, 8, F32)                     # nothing outside the rows is touched
        assert ws.status() == 1
        out, lse = attend(b, ws, q, 8, F32)          # not a row is written
        assert ws.status() == 1 and np.isnan(out).all() and np.isnan(lse).all()
    b.off = off
    b.upload()
    out, _ = attend(b, ws, q, 8, F32)
    assert ws.status() == 0 and np.array_equal(out, clean)
    ws.close()
    b.close()


@pytest.mark.parametrize("type_,ctype", [(F32, F32), (BF16, BF16)])
def test_offsets_beyond_32_bits(cpg, type_, ctype):
    """a pool whose pages lie 2^31 + elements apart: decode, a chunk, and the append"""
    b = Batch([(40, 1), (33, 33)], 1, 64, 16, ctype, spare=0).fill()
    stride = (1 << 31) // (4 if ctype == F32 else 2) * 2 // (2 if ctype == F32 else 1) + 4096
    eb = 4 if ctype == F32 else 2
    big = [C.DeviceBuffer(((b.n_pages - 1) * stride + b.page_stride) * eb) for _ in range(2)]
    for host, dev in zip((b.k, b.v), big):
        for p in range(b.n_pages):
            dev.upload(host[p * b.page_stride:(p + 1) * b.page_stride], p * stride * eb)
    b.upload()
    ws = Workspace(4, 1, 64)
    q = queries(b, 4, type_)
    small = attend(b, ws, q, 4, type_)
    held, b.page_stride = b.page_stride, stride
    keep = b.dev["k"], b.dev["v"]
    b.dev["k"], b.dev["v"] = big
    got = attend(b, ws, q, 4, type_)
    assert np.array_equal(got[0].view(np.uint8), small[0].view(np.uint8)) and np.array_equal(got[1], small[1])
    kn = np.random.default_rng(1).standard_normal((b.T, 64)).astype(np.float32)
    dk = C.to_device(to_type(kn, type_))
    C.check(C.lib().cpg_paged_append(ctypes.byref(b.cache()), ctypes.byref(b.batch()), None, type_, 0, None, 0,
                                     dk.ptr, 64, dk.ptr, 64, None, 0, ws.ptr), "append")
    C.sync()
    for s, (L, n) in enumerate(b.seqs):
        for i in range(n):
            j = L - n + i
            at = (int(b.pages[s, j // 16]) * stride + j % 16 * b.slot_stride) * eb
            for dev in big:
                row = dev.download(storage(ctype), 64, at)
                assert np.array_equal(row, to_type(kn[int(b.off[s]) + i], ctype))
    b.dev["k"], b.dev["v"] = keep
    b.page_stride = held
    for d in big + [dk]:
        d.close()
    ws.close()
    b.close()


# ---------------------------------------------------------------- append

def append64(x, gain, eps, table, pos, rot, adjacent):
    """heads (n, HD) in 64 bits: normed, turned"""
    x = x.copy()
    if gain is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * gain
    if rot:
        cs = table[pos]
        a, b = (x[:, 0:rot:2], x[:, 1:rot:2]) if adjacent else (x[:, :rot // 2], x[:, rot // 2:rot])
        ra, rb = a * cs[:, 0] - b * cs[:, 1], b * cs[:, 0] + a * cs[:, 1]
        y = x.copy()
        if adjacent:
            y[:, 0:rot:2], y[:, 1:rot:2] = ra, rb
        else:
            y[:, :rot // 2], y[:, rot // 2:rot] = ra, rb
        x = y
    return x


def do_append(b, H, type_, rot, adjacent, norm, in_place=False, pad=0, max_pos=None, seed=11):
    """runs cpg_paged_append and checks every query row and the whole pool; returns what it read"""
    KV, HD, T = b.KV, b.HD, b.T
    rng = np.random.default_rng(seed)
    row = (H + 2 * KV) * HD + pad
    x = to_type(rng.standard_normal((T, row)) * 1.5, type_)
    gains = (1 + 0.2 * rng.standard_normal((2, HD))).astype(np.float32) if norm else None
    max_pos = max_pos or int(max(b.len.max(), 1))
    ang = rng.uniform(0, 6.28, (max_pos, rot // 2)) if rot else np.zeros((1, 1))
    table = np.stack([np.cos(ang), np.sin(ang)], -1).astype(np.float32)
    dx, dt = C.to_device(x), C.to_device(table)
    dg = C.to_device(gains) if norm else None
    do = C.to_device(to_type(np.full((max(T, 1), max(H, 1) * HD), np.nan), type_))
    eb = x.itemsize
    R = C.PagedRope(dt.ptr, max_pos, rot, C.ROPE_ADJACENT if adjacent else C.ROPE_HALVES, dg and dg.ptr,
                    dg and dg.ptr + 4 * HD, 1e-6)
    ws = Workspace(max(H, KV), KV, HD)
    qo, ldqo = (dx.ptr, row) if in_place else (do.ptr, H * HD)
    C.check(C.lib().cpg_paged_append(ctypes.byref(b.cache()), ctypes.byref(b.batch()), ctypes.byref(R), type_, H,
                                     dx.ptr if H else None, row, dx.ptr + eb * H * HD, row,
                                     dx.ptr + eb * (H + KV) * HD, row, qo if H else None, ldqo, ws.ptr), "append")
    status = ws.status()
    if in_place:
        qgot = dx.download(storage(type_), T * row).reshape(T, row)[:, :H * HD].reshape(T, H, HD)
    else:
        qgot = do.download(storage(type_), max(T, 1) * max(H, 1) * HD)[:T * H * HD].reshape(T, H, HD)
    for d in (dx, dt, do) + ((dg,) if norm else ()):
        d.close()
    ws.close()
    return x, gains, table.transpose(0, 2, 1).astype(np.float64), qgot, status


def check_append(b, H, type_, rot, adjacent, norm, x, gains, table, qgot, skip=()):
    """skip: (s, i) of rows whose token must not have been stored"""
    KV, HD = b.KV, b.HD
    xv = values(x, type_)[:, :(H + 2 * KV) * HD].reshape(b.T, H + 2 * KV, HD)
    kw, vw = b.k.copy(), b.v.copy()
    # normed: 2 x 2^-24 sqrt(HD) + four roundings; turned: two products and a sum of two elements
    rel = (2.0 ** -24 * (2 * np.sqrt(HD) + 6) if norm else 0.0) + (2.0 ** -24 * 4 if rot else 0.0)

    def near(got, want, t):
        size = np.abs(want) + (np.abs(want).max() if rot else 0.0)
        # rounded to the type: half a step of the value, or of the smallest normal number
        tol = rel * size + HALF_STEP[t] * np.abs(want) * (1 + rel) + (2.0 ** -25 if t == F16 else 0.0)
        assert (np.abs(values(got, t) - want) <= tol).all(), np.abs(values(got, t) - want).max()

    kg, vg = b.pool()
    seen = np.zeros(b.T, bool)
    for s, (L, n) in enumerate(b.seqs):
        for i in range(n):
            t, p = int(b.off[s]) + i, L - n + i
            seen[t] = True
            if (s, i) in skip:
                if H:
                    assert np.isnan(values(qgot[t], type_)).all()
                continue
            pos = np.array([p])
            for h in range(H):
                near(qgot[t, h], append64(xv[t, h:h + 1], None if gains is None else gains[0].astype(float), 1e-6,
                                          table, pos, rot, adjacent)[0], type_)
            w = b.where(s, p)
            for h in range(KV):
                near(kg[w[h]], append64(xv[t, H + h:H + h + 1], None if gains is None else gains[1].astype(float),
                                        1e-6, table, pos, rot, adjacent)[0], b.ctype)
                assert np.array_equal(vg[w[h]], to_type(xv[t, H + KV + h], b.ctype))
            kg[w], vg[w] = kw[w], vw[w]
    # nothing else in the pool has changed, and rows of no sequence have no query
    assert np.array_equal(kg.view(np.uint8), kw.view(np.uint8))
    assert np.array_equal(vg.view(np.uint8), vw.view(np.uint8))
    return seen


APPENDS = [(4, 2, 64, 64, False, True), (8, 1, 128, 128, False, True), (2, 2, 96, 96, False, True),
           (6, 3, 192, 192, True, False), (1, 1, 256, 256, False, False), (5, 5, 128, 64, False, True),
           (4, 1, 96, 48, True, True), (32, 4, 128, 128, False, True), (4, 2, 64, 0, False, True),
           (4, 2, 64, 0, False, False), (3, 1, 256, 16, True, True), (0, 2, 128, 128, False, True),
           (0, 40, 64, 32, False, False), (70, 7, 64, 64, False, True)]


@pytest.mark.parametrize("type_,ctype", COMBOS)
@pytest.mark.parametrize("H,KV,HD,rot,adjacent,norm", APPENDS)
def test_append(cpg, type_, ctype, H, KV, HD, rot, adjacent, norm):
    say(f"append {NAMES[type_]}/{NAMES[ctype]} H={H} KV={KV} HD={HD} rot={rot} adjacent={adjacent} norm={norm}")
    b = Batch([(1, 1), (37, 5), (20, 0), (64, 33), (130, 1)], KV, HD, 16, ctype, by_head=H % 2 == 0,
              gap=8 * (HD % 3), T=45, first_row=2).upload()
    x, g, table, q, status = do_append(b, H, type_, rot, adjacent, norm, pad=8)
    assert status == 0
    seen = check_append(b, H, type_, rot, adjacent, norm, x, g, table, q)
    if H:
        assert np.isnan(values(q[~seen], type_)).all()
    b.close()


@pytest.mark.parametrize("page", [1, 4, 128])
def test_append_pages_and_in_place(cpg, page):
    b = Batch([(200, 150), (3, 3)], 2, 128, page, BF16).upload()
    x, g, table, q, status = do_append(b, 4, BF16, 128, False, True, in_place=True)
    assert status == 0
    check_append(b, 4, BF16, 128, False, True, x, g, table, q)
    b.close()


def test_append_many_sequences(cpg):
    """the search for a row's sequence over more than 64 and more than 4096 of them, many empty"""
    rng = np.random.default_rng(9)
    for S in (65, 130, 5000):
        seqs = [(int(n + rng.integers(0, 9)), int(n)) for n in rng.integers(0, 3, S)]
        b = Batch(seqs, 1, 64, 4, F32).upload()
        x, g, table, q, status = do_append(b, 1, F32, 64, False, False)
        assert status == 0
        check_append(b, 1, F32, 64, False, False, x, g, table, q)
        b.close()


def test_append_bad_rows(cpg):
    """positions before 0 and beyond the table, lengths beyond the pages: nothing is stored, the query
    is NaN, the status says so"""
    seqs = [(4, 6), (20, 3), (9, 2)]
    b = Batch(seqs, 2, 64, 16, F32).upload()
    x, g, table, q, status = do_append(b, 4, F32, 64, False, True, max_pos=19)
    assert status == 1
    check_append(b, 4, F32, 64, False, True, x, g, table, q, skip={(0, 0), (0, 1), (1, 2)})
    b.close()
    b = Batch(seqs, 2, 64, 16, F32)
    b.len[1] = b.max_pages * 16 + 1
    b.upload()
    x, g, table, q, status = do_append(b, 4, F32, 64, False, True, max_pos=64)
    assert status == 1
    check_append(b, 4, F32, 64, False, True, x, g, table, q, skip={(0, 0), (0, 1), (1, 0), (1, 1), (1, 2)})
    b.close()


def test_append_bad_page(cpg):
    b = Batch([(20, 1), (30, 1)], 2, 64, 16, F32)
    for bad in (-1, b.n_pages, 2 ** 31 - 1):
        b.pages[0, 1] = bad
        b.upload()
        k0 = b.pool()[0]
        x, g, table, q, status = do_append(b, 4, F32, 64, False, False)
        assert status == 1
        assert np.isfinite(q[:2]).all()              # the query needs no page
        kg = b.pool()[0]
        w = b.where(1, 29)
        assert np.isfinite(kg[w]).all()
        kg[w] = k0[w]
        assert np.array_equal(kg.view(np.uint32), k0.view(np.uint32))
    b.close()


# ---------------------------------------------------------------- together

def test_graph_replays_as_the_batch_moves(cpg):
    """append and attention captured once, replayed for steps whose lengths, pages and rows change on the
    device, against the same steps run eagerly"""
    H, KV, HD, S = 8, 2, 64, 5
    lens = np.array([3, 130, 17, 40, 0], np.int32)
    live = np.array([1, 1, 1, 1, 0])                 # a padded batch: sequence 4 brings nothing
    b = Batch([(200, n) for n in live], KV, HD, 16, F32, T=S).fill()
    b.len = lens.copy()
    b.upload()
    ws, rng = Workspace(H, KV, HD), np.random.default_rng(2)
    row = (H + 2 * KV) * HD
    ang = rng.uniform(0, 6.28, (200, HD // 2))
    table = C.to_device(np.stack([np.cos(ang), np.sin(ang)], -1).astype(np.float32))
    dx, dq, do = C.DeviceBuffer(S * row * 4), C.DeviceBuffer(S * H * HD * 4), C.DeviceBuffer(S * H * HD * 4)
    cache, batch = b.cache(), b.batch()
    R = C.PagedRope(table.ptr, 200, HD, C.ROPE_HALVES, None, None, 0.0)
    L = C.lib()

    def enqueue():
        C.check(L.cpg_paged_append(ctypes.byref(cache), ctypes.byref(batch), ctypes.byref(R), F32, H, dx.ptr, row,
                                   dx.ptr + 4 * H * HD, row, dx.ptr + 4 * (H + KV) * HD, row, dq.ptr, H * HD,
                                   ws.ptr), "append")
        C.check(L.cpg_paged_attn(ctypes.byref(cache), ctypes.byref(batch), F32, H, dq.ptr, H * HD, 0.0, 0, do.ptr,
                                 H * HD, None, ws.ptr), "attn")

    C.check(L.cpg_capture_begin(), "capture")
    enqueue()
    graph = L.cpg_capture_end()
    assert graph, C.last_error()
    for step in range(6):
        b.len = lens + live.astype(np.int32) * step
        if step == 3:                                # sequence 4 joins, sequence 0 leaves
            b.off = np.array([0, 0, 1, 2, 3, 4], np.int32)
            b.len[4] = 1
        elif step > 3:
            b.len[4] = step - 2
        b.dev["len"].upload(b.len)
        b.dev["off"].upload(b.off)
        x = rng.standard_normal((S, row)).astype(np.float32)
        before = b.pool()
        got = []
        for how in (lambda: C.check(L.cpg_graph_launch(graph), "launch"), enqueue):
            dx.upload(x)
            for d, a in zip(("k", "v"), before):
                b.dev[d].upload(a)
            do.zero()
            how()
            C.sync()
            got.append((do.download(np.float32, S * H * HD),) + b.pool())
        for a, e in zip(*got):
            assert np.array_equal(a.view(np.uint32), e.view(np.uint32)), step
        assert np.isfinite(got[0][0]).all() and np.abs(got[0][0]).max() > 0
    assert ws.status() == 0
    L.cpg_graph_destroy(graph)
    for d in (table, dx, dq, do):
        d.close()
    ws.close()
    b.close()


def test_two_graphs_over_one_workspace(cpg):
    """a graph of decode steps and one of prompts, with the same workspace, replayed in turn"""
    H, KV, HD = 8, 2, 128
    ws, L = Workspace(H, KV, HD), C.lib()
    made = []
    for seqs in ([(900, 1), (60, 1), (2500, 1)], [(700, 300), (64, 64), (1200, 90)]):
        b = Batch(seqs, KV, HD, 16, BF16).fill().upload()
        q = queries(b, H, BF16)
        want, _ = attend(b, ws, q, H, BF16)
        dq, do = C.to_device(to_type(q, BF16)), C.DeviceBuffer(b.T * H * HD * 2)
        cache, batch = b.cache(), b.batch()

        def enqueue():
            C.check(L.cpg_paged_attn(ctypes.byref(cache), ctypes.byref(batch), BF16, H, dq.ptr, H * HD, 0.0, 0,
                                     do.ptr, H * HD, None, ws.ptr), "attn")

        C.check(L.cpg_capture_begin(), "capture")
        enqueue()
        graph = L.cpg_capture_end()
        assert graph, C.last_error()
        made.append((b, dq, do, graph, want))
    for turn in range(4):
        for b, dq, do, graph, want in made:
            do.zero()
        for b, dq, do, graph, want in made + made:   # no synchronisation between them
            C.check(L.cpg_graph_launch(graph), "launch")
        C.sync()
        for b, dq, do, graph, want in made:
            got = do.download(np.uint16, b.T * H * HD).reshape(want.shape)
            assert np.array_equal(got, want), turn
    assert ws.status() == 0
    for b, dq, do, graph, want in made:
        L.cpg_graph_destroy(graph)
        for d in (dq, do, b):
            d.close()
    ws.close()


@pytest.mark.parametrize("type_,ctype", [(F32, F32), (BF16, BF16)])
def test_sequences_that_share_pages(cpg, type_, ctype):
    """a prefix held once by three sequences, and a page that a sequence has twice"""
    b = Batch([(200, 20), (180, 1), (170, 3), (96, 40)], 2, 64, 16, ctype).fill()
    b.pages[1, :8] = b.pages[2, :8] = b.pages[0, :8]
    b.pages[3, 3] = b.pages[3, 1]
    b.upload()
    ws = Workspace(8, 2, 64)
    q = queries(b, 8, type_)
    out, lse = attend(b, ws, q, 8, type_)
    assert ws.status() == 0
    compare(b, q, 8, type_, out, lse)
    ws.close()
    b.close()


@pytest.mark.parametrize("ctype", [F32, BF16])
def test_serving_steps_against_the_layer(cpg, ctype):
    """Two conversations served together through the paged cache (projection, append, attention, output
    projection: prompts first, then tokens of both at once, one prompt in two chunks) give what
    cpg_attn_forward gives for each alone over its own cache."""
    from tests.attn_helpers import DeviceAttn, attn_layer, inputs
    from tests.gpu_helpers import rel_err
    D, H, KV, HD, cap = 256, 4, 2, 64, 96
    a = attn_layer(D=D, H=H, KV=KV, HD=HD, enc=8)
    X = [inputs(D, 100, 60), inputs(D, 300, 60)]
    # (new tokens of conversation 0, of conversation 1) per step
    steps = [(20, 7), (1, 13), (1, 1), (1, 1), (0, 1), (9, 1), (1, 1)]
    dev = DeviceAttn(a, cap=cap, max_T=64)
    want = [np.zeros((0, D), np.float32)] * 2
    for c in range(2):
        dev.set_cache(np.zeros((cap, KV * HD)), np.zeros((cap, KV * HD)))
        pos, rows = 0, []
        for st in steps:
            if st[c]:
                rows.append(dev.forward(X[c][pos:pos + st[c]], pos))
                pos += st[c]
        want[c] = np.concatenate(rows)
    b = Batch([(cap, 0), (cap, 0)], KV, HD, 16, ctype)
    ws, L, row = Workspace(H, KV, HD), C.lib(), (H + 2 * KV) * HD
    R = C.PagedRope(dev.rope.ptr, cap, HD, C.ROPE_HALVES, dev.qn.ptr, dev.kn.ptr, a["eps"])
    pos, got = [0, 0], [[], []]
    b.upload()
    for st in steps:
        T = sum(st)
        x = C.to_device(np.concatenate([X[c][pos[c]:pos[c] + st[c]] for c in range(2)]))
        pos = [p + n for p, n in zip(pos, st)]
        b.off, b.len, b.T, b.seqs = np.array([0, st[0], T], np.int32), np.array(pos, np.int32), T, list(zip(pos, st))
        b.dev["off"].upload(b.off)
        b.dev["len"].upload(b.len)
        qkv, q, ao, out = (C.DeviceBuffer(T * n * 4) for n in (row, H * HD, H * HD, D))
        C.check(L.cpg_gemv_norm(8, dev.wqkv.ptr, D, row, x.ptr, T, dev.ln1.ptr, a["eps"], qkv.ptr), "qkv")
        C.check(L.cpg_paged_append(ctypes.byref(b.cache()), ctypes.byref(b.batch()), ctypes.byref(R), F32, H,
                                   qkv.ptr, row, qkv.ptr + 4 * H * HD, row, qkv.ptr + 4 * (H + KV) * HD, row,
                                   q.ptr, H * HD, ws.ptr), "append")
        C.check(L.cpg_paged_attn(ctypes.byref(b.cache()), ctypes.byref(b.batch()), F32, H, q.ptr, H * HD, 0.0, 0,
                                 ao.ptr, H * HD, None, ws.ptr), "attn")
        C.check(L.cpg_gemv(8, dev.wo.ptr, H * HD, D, ao.ptr, T, out.ptr), "wo")
        C.sync()
        o = out.download(np.float32, T * D).reshape(T, D)
        got[0].append(o[:st[0]])
        got[1].append(o[st[0]:])
        for d in (x, qkv, q, ao, out):
            d.close()
    assert ws.status() == 0
    # f32: both paths' sums in fp32; bf16: keys and values off by half a step each, a score by that
    # of |q||k| scale / sqrt(HD) of its terms, against outputs that average values of size 1
    tol = 2e-5 if ctype == F32 else 4 * HALF_STEP[BF16]
    for c in range(2):
        e = rel_err(np.concatenate(got[c]), want[c])
        say(f"conversation {c}: {e:.2e}")
        assert e <= tol
    ws.close()
    b.close()
    dev.close()


def test_workspace_geometry_refusals(cpg):
    b = Batch([(4, 1)], 2, 64, 16, F32).fill().upload()
    L = C.lib()
    for H, KV, HD in ((0, 1, 64), (4, 3, 64), (4, 0, 64), (4, 2, 80), (4, 2, 512), (-4, -2, 64), (1 << 20, 1, 64)):
        assert L.cpg_paged_ws_create(H, KV, HD) is None
    q = C.DeviceBuffer(8 * 64 * 4)
    for geom in ((8, 2, 64), (4, 4, 64), (4, 2, 128)):
        ws = Workspace(*geom)
        assert L.cpg_paged_attn(ctypes.byref(b.cache()), ctypes.byref(b.batch()), F32, 4, q.ptr, 256, 0.0, 0,
                                q.ptr, 256, None, ws.ptr) == -1
        assert "workspace" in C.last_error()
        assert L.cpg_paged_append(ctypes.byref(b.cache()), ctypes.byref(b.batch()), None, F32, 4, q.ptr, 256,
                                  q.ptr, 128, q.ptr, 128, q.ptr, 256, ws.ptr) == -1
        ws.close()
    q.close()
    b.close()
