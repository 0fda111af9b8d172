"""What the operators of the paged key/value cache are timed on.

A serving program keeps the keys and values of many sequences in pages of a common pool. Per layer
and step it makes two calls (include/cpg.h):

  append  cpg_paged_append: the new tokens' query, key and value heads as the projections leave
          them; the head norms and the position rotation are applied, keys and values go to their
          pages and the queries to a buffer;
  attn    cpg_paged_attn: the attention of the new tokens over everything their sequences hold.

A sequence of a case held `ctx` tokens before the call and brings `new` ones; both are spread over
the case's ranges. Widths are those of the configuration that the framework is built for (32 query
heads, 4 or 8 key/value heads of 128) and, in two cases and the drawn ones, other head layouts.
"""
import ctypes
import math

import torch

own = False

F32, F16, BF16 = "f32", "f16", "bf16"
TYPES = {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16}
EPS, THETA = 1e-6, 1e6


# ---------------------------------------------------------------- the cases

def _case(kind, act, cache, heads, page, S, ctx, new, window=0, by_head=False, norm=True, rot=None,
          adjacent=False, **more):
    H, KV, HD = heads
    c = dict(more, kind=kind, act=act, cache=cache, H=H, KV=KV, HD=HD, page=page, S=S, ctx_lo=ctx[0],
             ctx_hi=ctx[1], new_lo=new[0], new_hi=new[1], by_head=by_head)
    if kind == "attn":
        return dict(c, window=window)
    return dict(c, norm=norm, rot=HD if rot is None else rot, adjacent=adjacent)


def listed():
    q = (32, 4, 128)
    return [
        # one decoded token of one conversation
        _case("append", F32, F32, q, 16, 1, (200, 200), (1, 1), name="append_token"),
        # a decode batch, the cache in half the bytes
        _case("append", F32, BF16, q, 64, 64, (100, 2000), (1, 1), name="append_batch64"),
        # a whole chunk of a long prompt
        _case("append", F32, F32, q, 16, 1, (3584, 3584), (512, 512), name="append_chunk512"),
        # prompts of several requests, 16-bit activations, rotation of adjacent pairs in part of a head
        _case("append", BF16, BF16, (32, 8, 128), 32, 7, (0, 0), (300, 4000), norm=False, rot=64,
              adjacent=True, name="append_prompts"),
        # one token early in a conversation: what latency counts for
        _case("attn", F32, F32, q, 16, 1, (200, 200), (1, 1), name="attn_token_p200"),
        # a decode batch of conversations of every length
        _case("attn", F32, F32, q, 16, 16, (100, 2000), (1, 1), name="attn_batch16"),
        # one token far into a long document
        _case("attn", F32, BF16, q, 16, 1, (32767, 32767), (1, 1), name="attn_token_p32767"),
        # a full serving batch, 16-bit throughout
        _case("attn", BF16, BF16, (32, 8, 128), 16, 96, (500, 8000), (1, 1), name="attn_batch96"),
        # a short chat turn appended to its conversation
        _case("attn", F32, F32, q, 16, 1, (700, 700), (21, 21), name="attn_turn21"),
        # the last chunk of a prompt of 4096 tokens
        _case("attn", F32, F32, q, 16, 1, (3584, 3584), (512, 512), name="attn_chunk512"),
        # prompts of several requests from their first token, 16-bit throughout
        _case("attn", BF16, BF16, (32, 8, 128), 64, 3, (0, 0), (1500, 4500), name="attn_prompts"),
        # prompts' chunks and decoded tokens in one batch, a sliding window, heads of 64 with keys of
        # their own, pages laid out head by head
        _case("attn", F16, F16, (16, 16, 64), 32, 12, (50, 3000), (1, 300), window=1024, by_head=True,
              name="attn_mixed_window"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    act = rng.choice([F32, F32, F16, BF16])
    cache = rng.choice([F32, F16, BF16]) if act == F32 else act
    KV, G, HD = rng.choice([1, 2, 4, 4, 8]), rng.choice([1, 3, 4, 8, 8]), rng.choice([64, 96, 128, 128, 128, 256])
    heads, page = (KV * G, KV, HD), rng.choice([8, 16, 16, 32, 64, 128])
    by_head = rng.random() < 0.3
    if rng.random() < 0.35:
        S = _log_int(rng, 1, 64)
        hi = _log_int(rng, 1, max(1, 4000 // S)) if rng.random() < 0.6 else 1
        ctx = _log_int(rng, 1, 4000)
        return _case("append", act, cache, heads, page, S, (max(1, ctx // 8), ctx), (max(1, hi // 4), hi),
                     by_head=by_head, norm=rng.random() < 0.5, rot=rng.choice([HD, HD, HD // 2]),
                     adjacent=rng.random() < 0.3)
    window = _log_int(rng, 16, 4000) if rng.random() < 0.25 else 0
    form = rng.random()
    if form < 0.45:                              # decode batches
        S = _log_int(rng, 1, 96)
        ctx = _log_int(rng, 20, min(32767, 200000 // S))
        new = (1, 1)
    elif form < 0.7:                             # a chunk or a turn of one sequence
        S, n = 1, _log_int(rng, 2, 1500)
        ctx, new = _log_int(rng, 1, 6000), (n, n)
    else:                                        # ragged batches
        S = _log_int(rng, 2, 12)
        hi = _log_int(rng, 2, 2400 // S)
        ctx, new = _log_int(rng, 1, 4000), (1, hi)
    return _case("attn", act, cache, heads, page, S, (max(1, ctx // 8), ctx), new, window=window,
                 by_head=by_head)


def _spread(lo, hi, S, step):
    """S whole numbers over [lo, hi], even in their logarithm, in an order that is not sorted"""
    if lo == hi:
        return [lo] * S
    return [round(max(lo, 0.5) * (hi / max(lo, 0.5)) ** ((0.31 + (i + 1) * step) % 1.0)) for i in range(S)]


def _lengths(case):
    """(tokens held before the call, new tokens) of each sequence"""
    return (_spread(case["ctx_lo"], case["ctx_hi"], case["S"], 0.6180339887),
            _spread(case["new_lo"], case["new_hi"], case["S"], 0.7548776662))


# ---------------------------------------------------------------- inputs

class _State:
    pass


def _normal(g, *shape, sigma=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * sigma


def _angles(rot, positions):
    """the rotation table: (cos, sin) of every position and pair, in 32 bits"""
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    a = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * THETA ** (-2.0 * i / rot)
    return torch.stack([a.cos(), a.sin()], -1).float().contiguous()


def prepare(case, seed):
    s = _State()
    s.case = case
    S, H, KV, HD, P = (case[k] for k in ("S", "H", "KV", "HD", "page"))
    act, cache = TYPES[case["act"]], TYPES[case["cache"]]
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 13)
    ctx, new = _lengths(case)
    total = [c + n for c, n in zip(ctx, new)]
    s.T, s.max_new, s.max_len = sum(new), max(new), max(total)
    off = [0]
    for n in new:
        off.append(off[-1] + n)
    s.q_off = torch.tensor(off, dtype=torch.int32, device="cuda")
    s.len = torch.tensor(total, dtype=torch.int32, device="cuda")
    # pages handed out in a random order, as after a while of serving; unused entries are 0
    need = [-(-t // P) for t in total]
    s.max_pages = max(need)
    order = torch.randperm(sum(need) + 3, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(S, s.max_pages, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    s.pages, s.n_pages = table, sum(need) + 3
    # the pools, seen as (page, slot, head, dim) whichever of slot and head is outer in memory
    shape = (s.n_pages, KV, P, HD) if case["by_head"] else (s.n_pages, P, KV, HD)

    def pool(sigma):
        x = _normal(g, *shape, sigma=sigma).to(cache)
        return x.transpose(1, 2) if case["by_head"] else x

    s.k, s.v = pool(1.0), pool(0.9)
    if case["kind"] == "attn":
        s.q = _normal(g, s.T, H, HD).to(act)
        s.out = torch.empty(s.T, H, HD, dtype=act, device="cuda")
        s.lse = torch.empty(s.T, H, device="cuda")
    else:
        # the projections' output: q | k | v heads of each token, one row
        s.qkv = _normal(g, s.T, (H + 2 * KV) * HD, sigma=0.8).to(act)
        s.gain = 1.0 + _normal(g, 2, HD, sigma=0.1) if case["norm"] else None
        s.rope = _angles(case["rot"], s.max_len)
        s.out = torch.empty(s.T, H, HD, dtype=act, device="cuda")
    return s


# ---------------------------------------------------------------- one pass: plain

def _rows(s):
    """of each new token: its sequence, its place among the sequence's new tokens, its position"""
    t = torch.arange(s.T, dtype=torch.int32, device="cuda")
    seq = torch.searchsorted(s.q_off[1:], t, right=True)
    i = t - s.q_off[seq]
    return seq, i.long(), (s.len - (s.q_off[1:] - s.q_off[:-1]))[seq].long() + i


def _plain_append(s):
    c = s.case
    H, KV, HD, rot = c["H"], c["KV"], c["HD"], c["rot"]
    seq, _, pos = _rows(s)
    x = s.qkv.float().view(s.T, H + 2 * KV, HD)
    qk, v = x[:, :H + KV], x[:, H + KV:]
    if s.gain is not None:
        gain = s.gain[(torch.arange(H + KV, device="cuda") >= H).long()]
        qk = qk / (qk.square().mean(-1, keepdim=True) + EPS).sqrt() * gain
    cos, sin = s.rope[pos][:, None, :, 0], s.rope[pos][:, None, :, 1]
    a, b = (qk[..., 0:rot:2], qk[..., 1:rot:2]) if c["adjacent"] else (qk[..., :rot // 2], qk[..., rot // 2:rot])
    ra, rb = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([ra, rb], -1).flatten(-2) if c["adjacent"] else torch.cat([ra, rb], -1)
    qk = torch.cat([turned, qk[..., rot:]], -1)
    page, slot = s.pages[seq, pos // c["page"]].long(), pos % c["page"]
    s.k[page, slot] = qk[:, H:].to(s.k.dtype)
    s.v[page, slot] = v.to(s.v.dtype)
    return {"q": qk[:, :H].to(s.out.dtype), "k": s.k, "v": s.v}


def _plain_attn(s):
    c = s.case
    S, H, KV, HD, P = (c[k] for k in ("S", "H", "KV", "HD", "page"))
    N, L, G = s.max_new, s.max_len, c["H"] // c["KV"]
    seq, place, _ = _rows(s)
    new = s.q_off[1:] - s.q_off[:-1]
    # keys and values of every sequence, (S, KV, L, HD); queries (S, KV, N * G, HD)
    j = torch.arange(L, device="cuda")
    page, slot = s.pages[:, j // P].long(), (j % P).expand(S, L)
    k = s.k[page, slot].float().transpose(1, 2).contiguous()
    v = s.v[page, slot].float().transpose(1, 2).contiguous()
    i = torch.arange(N, device="cuda")
    row = (s.q_off[:-1, None] + i).clamp(max=s.T - 1).long()
    q = s.q[row].float().view(S, N, KV, G, HD).transpose(1, 2).reshape(S, KV, N * G, HD)
    pos = ((s.len - new)[:, None] + i)[:, :, None]
    seen = (j <= pos) & (j < s.len[:, None, None])
    if c["window"]:
        seen &= j > pos - c["window"]
    x = torch.matmul(q, k.transpose(2, 3).contiguous()).view(S, KV, N, G, L) / math.sqrt(HD)
    x = x.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = x.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(S, KV, N * G, L), v).view(S, KV, N, G, HD) / total
    lse = (total.log() + top).squeeze(-1)
    return {"out": o[seq, :, place].reshape(s.T, H, HD).to(s.out.dtype),
            "lse": lse[seq, :, place].reshape(s.T, H)}


# ---------------------------------------------------------------- one pass: the framework's calls

_kept = {}


def _workspace(C, H, KV, HD):
    """the workspace that a program keeps for its layers' attention"""
    if (H, KV, HD) not in _kept:
        C.init(0)
        ws = C.lib().cpg_paged_ws_create(H, KV, HD)
        if not ws:
            raise C.CPGError(C.last_error())
        _kept[H, KV, HD] = ws
    return _kept[H, KV, HD]


def _own(s):
    import cachepotato_amd as C
    c = s.case
    H, KV, HD, T = c["H"], c["KV"], c["HD"], s.T
    ws = _workspace(C, H, KV, HD)
    kind = {F32: C.T_F32, F16: C.T_F16, BF16: C.T_BF16}
    ps, ss, hs, _ = s.k.stride()
    cache = C.PagedCache(KV, HD, kind[c["cache"]], c["page"], s.n_pages, ps, ss, hs, s.k.data_ptr(),
                         s.v.data_ptr())
    batch = C.PagedBatch(c["S"], T, s.max_new, s.max_pages, s.pages.data_ptr(), s.q_off.data_ptr(),
                         s.len.data_ptr())
    if c["kind"] == "attn":
        C.check(C.lib().cpg_paged_attn(ctypes.byref(cache), ctypes.byref(batch), kind[c["act"]], H,
                                       s.q.data_ptr(), H * HD, 0.0, c["window"], s.out.data_ptr(),
                                       H * HD, s.lse.data_ptr(), ws), "cpg_paged_attn")
        return {"out": s.out, "lse": s.lse}
    row, x, size = (H + 2 * KV) * HD, s.qkv.data_ptr(), s.qkv.element_size()
    gain = s.gain.data_ptr() if s.gain is not None else None
    turn = C.PagedRope(s.rope.data_ptr(), s.rope.shape[0], c["rot"],
                       C.ROPE_ADJACENT if c["adjacent"] else C.ROPE_HALVES, gain,
                       gain and gain + 4 * HD, EPS)
    C.check(C.lib().cpg_paged_append(ctypes.byref(cache), ctypes.byref(batch), ctypes.byref(turn),
                                     kind[c["act"]], H, x, row, x + size * H * HD, row,
                                     x + size * (H + KV) * HD, row, s.out.data_ptr(), H * HD, ws),
            "cpg_paged_append")
    return {"q": s.out, "k": s.k, "v": s.v}


def run(s):
    if own:
        return _own(s)
    return _plain_append(s) if s.case["kind"] == "append" else _plain_attn(s)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    H, KV, HD, P = (case[k] for k in ("H", "KV", "HD", "page"))
    size = {F32: 4, F16: 2, BF16: 2}
    a, b = size[case["act"]], size[case["cache"]]
    ctx, new = _lengths(case)
    T = sum(new)
    tables = 4.0 * (sum(-(-(c + n) // P) for c, n in zip(ctx, new)) + 2 * case["S"])
    if case["kind"] == "append":
        return {"bytes": T * ((2 * H + 2 * KV) * HD * a + 2 * KV * HD * b + 4 * case["rot"]) + tables,
                "flops": T * (H + KV) * (3.0 * case["rot"] + (4.0 * HD if case["norm"] else 0.0))}
    W = case["window"] or 1 << 30
    keys = sum(c + n - max(0, c + 1 - W) for c, n in zip(ctx, new))
    pairs = sum(sum(min(p, W) for p in range(c + 1, c + n + 1)) for c, n in zip(ctx, new))
    return {"bytes": 2.0 * KV * HD * b * keys + T * H * (2.0 * HD * a + 4) + tables,
            "flops": 4.0 * H * HD * pairs}


# ---------------------------------------------------------------- the same in 64 bits

def _sequence(s, i):
    """the rows of sequence i's new tokens, its length, and where its tokens are"""
    lo, hi, n = int(s.q_off[i]), int(s.q_off[i + 1]), int(s.len[i])
    at = [(int(p), k) for p in s.pages[i].tolist() for k in range(s.case["page"])][:n]
    at = torch.tensor(at, device="cuda").T
    return lo, hi, n, at[0], at[1]


def _exact_append(s):
    c = s.case
    H, KV, HD, r = c["H"], c["KV"], c["HD"], c["rot"]
    k, v = s.k.double(), s.v.double()
    q = torch.empty(s.T, H, HD, dtype=torch.float64, device="cuda")
    for i in range(c["S"]):
        lo, hi, n, page, slot = _sequence(s, i)
        heads = s.qkv[lo:hi].double().view(hi - lo, -1, HD).split([H, KV, KV], 1)
        turn = torch.view_as_complex(s.rope[n - (hi - lo):n].double())[:, None]
        done = []
        for x, gain in zip(heads[:2], (0, 1)):
            if s.gain is not None:
                x = x * s.gain[gain].double() * (x.pow(2).sum(-1, keepdim=True) / HD + EPS).rsqrt()
            x = x.clone()
            pairs = x[..., :r].unflatten(-1, (r // 2, 2) if c["adjacent"] else (2, r // 2))
            if not c["adjacent"]:
                pairs = pairs.transpose(-1, -2)
            z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
            x[..., :r] = (z if c["adjacent"] else z.transpose(-1, -2)).flatten(-2)
            done.append(x)
        q[lo:hi] = done[0]
        page, slot = page[n - (hi - lo):], slot[n - (hi - lo):]
        k[page, slot], v[page, slot] = done[1], heads[2]
    return {"q": q, "k": k, "v": v}


def _exact_attn(s):
    c = s.case
    H, KV, HD = c["H"], c["KV"], c["HD"]
    G = H // KV
    out = torch.empty(s.T, H, HD, dtype=torch.float64, device="cuda")
    lse = torch.empty(s.T, H, dtype=torch.float64, device="cuda")
    for i in range(c["S"]):
        lo, hi, n, page, slot = _sequence(s, i)
        behind = torch.arange(n - (hi - lo), n, device="cuda")[:, None] - torch.arange(n, device="cuda")
        hidden = (behind < 0) | (behind >= c["window"]) if c["window"] else behind < 0
        for h in range(KV):
            k, v = s.k[page, slot, h].double(), s.v[page, slot, h].double()
            for e in range(h * G, h * G + G):
                x = s.q[lo:hi, e].double() @ k.T * HD ** -0.5
                x.masked_fill_(hidden, -math.inf)
                lse[lo:hi, e] = x.logsumexp(-1)
                out[lo:hi, e] = x.softmax(-1) @ v
    return {"out": out, "lse": lse}


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_append(s) if case["kind"] == "append" else _exact_attn(s)
