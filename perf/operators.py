"""Serving many requests over one paged key/value cache: what its operators are measured on.

Four operators, each through its C entry point on device pointers:

* ``plan``       ``ptmi_paged_plan_dev``: block tables and slot maps from request lengths;
* ``store``      ``ptmi_paged_store_dev``: new q and k rows rotated, k and v written into their pages;
* ``attention``  ``ptmi_paged_attention_dev``: attention of each request's new tokens over its pages;
* ``sample``     ``ptmi_sample_dev``: one token per row of logits from given random numbers.

With ``own`` false the same results come from elementary torch operations.  torch supplies device
memory; it is imported before the package so that both use one HIP runtime.
"""
import ctypes
import math
import random

import torch

own = False

DEV = "cuda"


def listed():
    return [
        # The bookkeeping of one decode step of a few requests: the smallest call, pure latency.
        dict(name="plan_decode", op="plan", requests=16, new_lo=1, new_hi=1, past_lo=1, past_hi=1023, ended=0.0, page=16, lens=1),
        # A busy server's step: decodes, prompt chunks, requests that ended and idle ones.
        dict(name="plan_mixed", op="plan", requests=1021, new_lo=0, new_hi=96, past_lo=0, past_hi=4000, ended=0.1, page=16, lens=2),
        # One layer's keys and values of a decode step, 110M heads.
        dict(name="store_decode", op="store", rows=64, heads=12, kv_heads=12, head_dim=64, page=16, cache="f32"),
        # Prompt chunks of many requests, grouped heads, a 16-bit cache: the largest store.
        dict(name="store_prompt", op="store", rows=8190, heads=32, kv_heads=8, head_dim=128, page=64, cache="bf16"),
        # One short 15M request, one token: the latency of a small decode.
        dict(name="attn_one_15m", op="attention", requests=1, new_lo=1, new_hi=1, past_lo=37, past_hi=37, heads=6, kv_heads=6, head_dim=48,
             page=16, cache="f32", lens=3),
        # 64 110M requests anywhere in their context, one token each: ordinary decode, a stream of keys and values.
        dict(name="attn_decode_110m", op="attention", requests=64, new_lo=1, new_hi=1, past_lo=1, past_hi=1023, heads=12, kv_heads=12, head_dim=64,
             page=16, cache="f32", lens=4),
        # Two answers to very long documents, grouped heads and a 16-bit cache: few rows over a long axis.
        dict(name="attn_long", op="attention", requests=2, new_lo=1, new_hi=1, past_lo=70001, past_hi=131001, heads=32, kv_heads=8, head_dim=128,
             page=64, cache="bf16", lens=5),
        # Prompt chunks of 110M heads behind contexts of several chunks: the largest products.
        dict(name="attn_chunk_110m", op="attention", requests=16, new_lo=512, new_hi=512, past_lo=0, past_hi=3584, heads=12, kv_heads=12, head_dim=64,
             page=16, cache="f32", lens=6),
        # Chunks and single tokens together, sizes that divide by nothing, pages that end inside every tile.
        dict(name="attn_ragged", op="attention", requests=7, new_lo=1, new_hi=701, past_lo=0, past_hi=2003, heads=20, kv_heads=4, head_dim=80,
             page=24, cache="bf16", lens=7),
        # One request's next token from the stories vocabulary: latency.
        dict(name="sample_one", op="sample", rows=1, vocab=32000),
        # A batch of requests, each with its own parameters.
        dict(name="sample_batch", op="sample", rows=64, vocab=32000),
        # Many rows of a vocabulary that divides by nothing (no row but the first starts on 16 bytes).
        dict(name="sample_ragged", op="sample", rows=509, vocab=50259),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("plan", "store", "attention", "attention", "attention", "sample"))
    lens = rng.randrange(1 << 30)
    page = rng.choice((8, 16, 16, 24, 32, 64, 100))
    if op == "plan":
        top = _log(rng, 1, 96)
        return dict(op=op, requests=_log(rng, 1, 1021), new_lo=rng.choice((0, 1)), new_hi=top, past_lo=0, past_hi=_log(rng, 16, 4000),
                    ended=rng.choice((0.0, 0.1, 0.3)), page=rng.choice((8, 16, 16, 24, 32, 64)), lens=lens)
    if op == "sample":
        return dict(op=op, rows=_log(rng, 1, 500), vocab=rng.choice((32000, _log(rng, 2000, 50259))))
    kv = rng.choice((1, 2, 4, 6, 8, 12))
    group = rng.choice((1, 1, 2, 4, 5, 8)) if kv <= 4 else rng.choice((1, 1, 2, 3))
    hd = rng.choice((32, 48, 64, 64, 80, 96, 128, 36))
    cache = rng.choice(("f32", "f32", "bf16"))
    heads = kv * group
    if op == "store":
        rows = min(_log(rng, 1, 8000), max(1, (8000 * 48 * 128) // ((heads + 2 * kv) * hd)))
        return dict(op=op, rows=rows, heads=heads, kv_heads=kv, head_dim=hd, page=page, cache=cache)
    while True:
        kind = rng.choice(("decode", "chunk", "mixed"))
        s = _log(rng, 1, 64)
        past = _log(rng, 8, 100000 if kind == "decode" else 4000)
        new = 1 if kind == "decode" else _log(rng, 2, 700)
        case = dict(op=op, requests=s, new_lo=1 if kind == "mixed" else max(1, new - new // 8), new_hi=new,
                    past_lo=past // rng.choice((1, 2, 8)), past_hi=past,
                    heads=heads, kv_heads=kv, head_dim=hd, page=page, cache=cache, lens=lens)
        # The plain form pads every request to the longest.
        if s * (past + new) * kv * hd <= 2.4e8 and s * heads * new * (past + new) <= 3e8 and _attention_flops(case) <= 5e10:
            return case


# ── what a user's program has in hand ────────────────────────────────────

def _lengths(case):
    """(past, new) of each request: part of the case, not of the seed (-1 new: the request has ended)."""
    r = random.Random(case["lens"])
    past, new = [], []
    for _ in range(case["requests"]):
        past.append(r.randint(case["past_lo"], case["past_hi"]))
        new.append(-1 if r.random() < case.get("ended", 0.0) else r.randint(case["new_lo"], case["new_hi"]))
    return past, new


def _pages(n, page):
    return -(-n // page)


def _gen(seed):
    return torch.Generator(DEV).manual_seed(seed)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _table(case, seed, extra=0):
    """Shuffled pages for every request's tokens: (block table, the pages that are left, number of pages)."""
    past, new = _lengths(case)
    page = case["page"]
    need = [_pages(p + max(0, n) * extra, page) for p, n in zip(past, new)]
    width = max(1, max(_pages(p + max(0, n), page) for p, n in zip(past, new)))
    spare = sum(_pages(p + max(0, n), page) - _pages(p, page) for p, n in zip(past, new)) + 5
    total = sum(need) + spare
    order = torch.randperm(total, generator=_gen(seed), device=DEV).int()
    rows = torch.arange(width, device=DEV)[None, :].expand(len(need), width)
    start = torch.tensor([0] + need, device=DEV).cumsum(0)[:-1, None]
    used = rows < torch.tensor(need, device=DEV)[:, None]
    table = torch.where(used, order[(start + rows).clamp(max=total - 1)], -1).int().contiguous()
    return table, order[sum(need):], total


def _library():
    import pitorch_amd as pa
    return pa.load_ptmi(), pa._ffi.check, pa


def _cache_shape(case, n_pages):
    return (n_pages, case["page"], case["kv_heads"], case["head_dim"])


def _pages_struct(pa, s, case):
    """The description of the cache that a program keeps."""
    k = s["k"]
    return pa.Pages(k.data_ptr(), s["v"].data_ptr(), pa.BF16 if case["cache"] == "bf16" else pa.F32, k.shape[0], k.shape[1], k.shape[2],
                    k.shape[3], k.stride(0), k.stride(1), k.stride(2))


def prepare(case, seed):
    op, g = case["op"], _gen(seed)
    s = dict(case=case)
    if own:
        s["L"], s["check"], s["pa"] = _library()
    if op == "plan":
        past, new = _lengths(case)
        s["table"], free, n_pages = _table(case, seed)
        rows = sum(max(0, n) for n in new)
        s.update(past=_ints(past), fresh=_ints(new), n_pages=n_pages, max_rows=rows + 3)
        s["pool"] = torch.cat((free, torch.full((n_pages - len(free) + 1,), -1, dtype=torch.int32, device=DEV)))
        s["count"] = _ints([len(free)])
        S = len(past)
        s["out"] = dict(kv_len=_ints([0] * S), left=_ints([0]), row_start=_ints([0] * (S + 1)), row_pos=_ints([0] * s["max_rows"]),
                        row_slot=_ints([0] * s["max_rows"]), status=_ints([0]), table=s["table"], pool=s["pool"])
    elif op == "sample":
        rows, V = case["rows"], case["vocab"]
        r = random.Random(seed)
        # Logits as a language model gives them: a broad bulk and a few likely tokens.
        x = torch.randn(rows, V, generator=g, device=DEV) * 2.0
        x += 9.0 * torch.rand(rows, V, generator=g, device=DEV).pow(200.0)
        s["logits"] = x
        s["temperature"] = torch.tensor([r.choice((0.0, 0.7, 1.0, 1.0, 1.3)) if rows > 1 else 0.8 for _ in range(rows)], device=DEV)
        s["top_k"] = _ints([r.choice((0, 0, 20, 50, 400)) if rows > 1 else 0 for _ in range(rows)])
        s["top_p"] = torch.tensor([r.choice((1.0, 0.9, 0.95, 0.5)) if rows > 1 else 0.9 for _ in range(rows)], device=DEV)
        s["min_p"] = torch.tensor([r.choice((0.0, 0.0, 0.05)) if rows > 1 else 0.0 for _ in range(rows)], device=DEV)
        s["u"] = torch.rand(rows, generator=g, device=DEV)
        s["token"] = _ints([0] * rows)
    else:
        H, KV, hd, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
        dt = torch.bfloat16 if case["cache"] == "bf16" else torch.float32
        if op == "store":
            rows = case["rows"]
            n_pages = _pages(rows, page) + 3
            # Each row's own slot in shuffled pages, positions anywhere in a context; two padding rows at the end.
            order = torch.randperm(n_pages * page, generator=g, device=DEV)[:rows].int()
            s["slot"] = torch.where(torch.arange(rows, device=DEV) < max(1, rows - 2), order, -1).int()
            s["pos"] = torch.randint(0, 4096, (rows,), generator=g, device=DEV, dtype=torch.int32)
            i = torch.arange(0, hd, 2, device=DEV, dtype=torch.float64)
            a = torch.arange(4096, device=DEV, dtype=torch.float64)[:, None] * torch.exp(-math.log(10000.0) * i / hd)
            s["rope"] = torch.stack((torch.cos(a), torch.sin(a)), -1).float().contiguous()
            s["qkv"] = torch.randn(rows, (H + 2 * KV) * hd, generator=g, device=DEV)
            s["q_out"] = torch.zeros(rows, H * hd, device=DEV)
            s["k"], s["v"] = (torch.zeros(_cache_shape(case, n_pages), device=DEV, dtype=dt) for _ in range(2))
        else:
            past, new = _lengths(case)
            s["table"], _, n_pages = _table(case, seed, extra=1)
            s["k"], s["v"] = (torch.randn(_cache_shape(case, n_pages), generator=g, device=DEV, dtype=torch.float32).to(dt) for _ in range(2))
            s["kv_len"] = _ints([p + n for p, n in zip(past, new)])
            s["row_start"] = _ints([sum(new[:i]) for i in range(len(new) + 1)])
            s["rows"], s["max_new"] = sum(new), max(new)
            s["q"] = torch.randn(s["rows"], H * hd, generator=g, device=DEV) * 1.5
            s["out"] = torch.zeros(s["rows"], H * hd, device=DEV)
        if own:
            s["pages"] = _pages_struct(s["pa"], s, case)
            s["ref"] = ctypes.byref(s["pages"])
            if op == "attention":
                n = s["L"].ptmi_paged_attention_work(s["ref"], H, s["max_new"])
                s["work"] = torch.empty(max(n, 16), dtype=torch.uint8, device=DEV)
    torch.cuda.synchronize()
    return s


# ── one pass ─────────────────────────────────────────────────────────────

def run(s):
    case = s["case"]
    op = case["op"]
    if not own:
        return dict(plan=_plain_plan, store=_plain_store, attention=_plain_attention, sample=_plain_sample)[op](s)
    L, check = s["L"], s["check"]
    if op == "plan":
        o = s["out"]
        check(L.ptmi_paged_plan_dev(s["past"].data_ptr(), s["fresh"].data_ptr(), case["requests"], s["pool"].data_ptr(), s["count"].data_ptr(),
                                    s["n_pages"], case["page"], s["table"].data_ptr(), s["table"].shape[1], o["kv_len"].data_ptr(),
                                    o["left"].data_ptr(), o["row_start"].data_ptr(), o["row_pos"].data_ptr(), o["row_slot"].data_ptr(),
                                    s["max_rows"], o["status"].data_ptr(), None))
        return o
    if op == "sample":
        x = s["logits"]
        check(L.ptmi_sample_dev(x.data_ptr(), x.stride(0), x.shape[0], x.shape[1], s["temperature"].data_ptr(), s["top_k"].data_ptr(),
                                s["top_p"].data_ptr(), s["min_p"].data_ptr(), s["u"].data_ptr(), s["token"].data_ptr(), None))
        return s["token"]
    H, KV, hd = case["heads"], case["kv_heads"], case["head_dim"]
    if op == "store":
        x = s["qkv"]
        q, ld = x.data_ptr(), x.stride(0)
        check(L.ptmi_paged_store_dev(s["ref"], q, ld, s["q_out"].data_ptr(), H * hd, H, q + 4 * H * hd, q + 4 * (H + KV) * hd, ld,
                                     s["pos"].data_ptr(), s["slot"].data_ptr(), x.shape[0], s["rope"].data_ptr(), s["rope"].shape[0], None))
        return dict(q=s["q_out"], k=s["k"], v=s["v"])
    check(L.ptmi_paged_attention_dev(s["ref"], s["table"].data_ptr(), s["table"].shape[1], s["row_start"].data_ptr(), s["kv_len"].data_ptr(),
                                     case["requests"], s["max_new"], s["q"].data_ptr(), H * hd, s["out"].data_ptr(), H * hd, s["rows"], H,
                                     hd ** -0.5, s["work"].data_ptr(), s["work"].numel(), None))
    return s["out"]


# ── the plain forms ──────────────────────────────────────────────────────

def _before(n):
    """Exclusive running sums."""
    return torch.cumsum(n, 0) - n


def _plain_plan(s):
    case, P = s["case"], s["case"]["page"]
    past, fresh, table, pool = (s[k].long() for k in ("past", "fresh", "table", "pool"))
    W, rows, count = table.shape[1], s["max_rows"], s["count"].long()
    ended = fresh < 0
    new = fresh.clamp(min=0)
    old_pages = (past + P - 1) // P
    kv = torch.where(ended, 0, past + new)
    take = torch.where(ended, 0, (kv + P - 1) // P - old_pages)
    give = torch.where(ended, old_pages, 0)
    col = torch.arange(W, device=DEV)[None, :]
    # The ended requests' pages go on top of the pool, in order (others write its last, spare place).
    at = torch.where(col < give[:, None], count + _before(give)[:, None] + col, pool.numel() - 1)
    pool = pool.scatter(0, at.reshape(-1), table.reshape(-1))
    pool[-1] = -1
    top = count + give.sum()
    j = col - old_pages[:, None]
    fetched = pool[(top - 1 - (_before(take)[:, None] + j)).clamp(0, s["n_pages"] - 1)]
    table = torch.where((j >= 0) & (j < take[:, None]), fetched, table)
    start = torch.cat((torch.zeros(1, dtype=torch.long, device=DEV), torch.cumsum(new, 0)))
    r = torch.arange(rows, device=DEV)
    live = r < start[-1]
    req = torch.searchsorted(start[1:], r, right=True).clamp(max=len(past) - 1)
    pos = past[req] + r - start[req]
    slot = table[req, (pos // P).clamp(0, W - 1)] * P + pos % P
    status = (take.sum() > top).int() + 2 * (((kv + P - 1) // P) > W).any().int() + 4 * (start[-1] > rows).int()
    return dict(kv_len=kv.int(), left=(top - take.sum()).int(), row_start=start.int(), row_pos=torch.where(live, pos, -1).int(),
                row_slot=torch.where(live, slot, -1).int(), status=status.reshape(1).int(), table=table.int(), pool=pool.int())


def _turn(x, cs):
    """Rotates the pairs (2i, 2i+1) of [rows, heads, head_dim] by the rows' (cos, sin)."""
    u, v = x[..., 0::2], x[..., 1::2]
    c, n = cs[:, None, :, 0], cs[:, None, :, 1]
    return torch.stack((u * c - v * n, u * n + v * c), -1).flatten(-2)


def _plain_store(s):
    case = s["case"]
    H, KV, hd = case["heads"], case["kv_heads"], case["head_dim"]
    rows = s["qkv"].shape[0]
    x = s["qkv"].view(rows, H + 2 * KV, hd)
    live = (s["slot"] >= 0).nonzero()[:, 0]
    cs = s["rope"][s["pos"].long()]
    qk = _turn(x[:, :H + KV], cs)
    slot = s["slot"][live].long()
    s["q_out"].view(rows, H, hd)[live] = qk[live, :H]
    s["k"].view(-1, KV, hd)[slot] = qk[live, H:].to(s["k"].dtype)
    s["v"].view(-1, KV, hd)[slot] = x[live, H + KV:].to(s["v"].dtype)
    return dict(q=s["q_out"], k=s["k"], v=s["v"])


def _plain_attention(s):
    case = s["case"]
    S, H, KV, hd, P = case["requests"], case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    kv_len, start = s["kv_len"].long(), s["row_start"].long()
    n = start[1:] - start[:-1]
    N, W = s["max_new"], s["table"].shape[1]
    T = W * P
    # Every request padded to the longest: keys and values [S, KV, T, hd], queries [S, KV, G*N, hd].
    flat = s["table"].clamp(min=0).long().reshape(-1)
    k, v = (s[t].index_select(0, flat).float().view(S, T, KV, hd).transpose(1, 2).contiguous() for t in ("k", "v"))
    i = torch.arange(N, device=DEV)
    row = (start[:-1, None] + i).clamp(max=s["rows"] - 1)
    q = s["q"].view(-1, KV, H // KV, hd)[row].permute(0, 2, 3, 1, 4).reshape(S, KV, -1, hd).contiguous()
    pos = kv_len[:, None] - n[:, None] + i
    seen = (torch.arange(T, device=DEV) <= pos[..., None]) & (i < n[:, None])[..., None]
    w = torch.matmul(q, k.transpose(2, 3)).view(S, KV, H // KV, N, T).mul_(hd ** -0.5)
    w.masked_fill_(~seen[:, None, None], -math.inf)
    m = w.amax(-1, keepdim=True)
    w.sub_(torch.where(m == -math.inf, 0.0, m)).exp_()
    total = w.sum(-1, keepdim=True)
    o = torch.matmul(w.view(S, KV, -1, T), v).view(S, KV, H // KV, N, hd) / torch.where(total == 0, 1.0, total)
    o = o.permute(0, 3, 1, 2, 4).reshape(S, N, H * hd)
    return o[i < n[:, None]]


def _plain_sample(s):
    x = torch.where(s["logits"].isnan(), -math.inf, s["logits"])
    T = s["temperature"].double()[:, None]
    sorted_x, order = torch.sort(x, dim=1, descending=True, stable=True)
    top = sorted_x[:, :1].double()
    z = (sorted_x.double() - top) / torch.where(T > 0, T, 1.0)
    w = torch.where(sorted_x == sorted_x[:, :1], 1.0, torch.exp(z))       # (an infinite maximum: its equals)
    V = x.shape[1]
    rank = torch.arange(V, device=DEV)[None, :]
    k = torch.where(s["top_k"] > 0, s["top_k"], V)[:, None]
    w = torch.where((rank < torch.where(T > 0, k, 1)) & (w >= s["min_p"].double()[:, None]), w, 0.0)
    c = torch.cumsum(w, 1)
    before = torch.cat((torch.zeros_like(c[:, :1]), c[:, :-1]), 1)
    p = s["top_p"].double()[:, None]
    w = torch.where((before < p * c[:, -1:]) | (p >= 1) | (rank == 0), w, 0.0)
    c = torch.cumsum(torch.zeros_like(w).scatter_(1, order, w), 1)
    token = (c <= s["u"].double()[:, None] * c[:, -1:]).sum(1)
    return torch.where(top[:, 0] == -math.inf, -1, token).int()


# ── what a pass cannot do without ────────────────────────────────────────

def _seen(case):
    past, new = _lengths(case)
    return sum(n * p + n * (n + 1) // 2 for p, n in zip(past, new))


def _attention_flops(case):
    return 4.0 * case["head_dim"] * case["heads"] * _seen(case)


def work(case):
    op = case["op"]
    if op == "plan":
        past, new = _lengths(case)
        rows = sum(max(0, n) for n in new)
        moved = sum(_pages(p, case["page"]) if n < 0 else _pages(p + n, case["page"]) - _pages(p, case["page"]) for p, n in zip(past, new))
        return dict(bytes=4.0 * (4 * len(past) + 2 * moved + 2 * rows + 8), flops=0.0)
    if op == "sample":
        return dict(bytes=4.0 * case["rows"] * (case["vocab"] + 6), flops=2.0 * case["rows"] * case["vocab"])
    H, KV, hd = case["heads"], case["kv_heads"], case["head_dim"]
    size = 2.0 if case["cache"] == "bf16" else 4.0
    if op == "store":
        rows = case["rows"]
        return dict(bytes=rows * (4.0 * (2 * H + 2 * KV) * hd + size * 2 * KV * hd + 8.0 + 4.0 * hd), flops=3.0 * rows * (H + KV) * hd)
    past, new = _lengths(case)
    tokens = sum(p + n for p, n in zip(past, new))
    return dict(bytes=size * 2 * tokens * KV * hd + 8.0 * sum(new) * H * hd, flops=_attention_flops(case))


# ── the same results in 64 bits ──────────────────────────────────────────

def exact(case, seed):
    if case["op"] in ("plan", "sample"):            # whole numbers
        return None
    s = prepare(case, seed)
    H, KV, hd = case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "store":
        rows = case["rows"]
        q, k, v = (t.double() for t in s["qkv"].split((H * hd, KV * hd, KV * hd), 1))
        out = []
        angle = torch.view_as_complex(s["rope"].double())[s["pos"].long()]
        for x, heads in ((q, H), (k, KV)):
            z = torch.view_as_complex(x.reshape(rows, heads, hd // 2, 2).contiguous()) * angle[:, None]
            out.append(torch.view_as_real(z).reshape(rows, heads * hd))
        got = dict(q=s["q_out"].double(), k=s["k"].double(), v=s["v"].double())
        at = s["slot"].long()
        got["q"] = out[0] * (at >= 0)[:, None]
        for name, x in (("k", out[1]), ("v", v)):
            got[name].view(-1, KV * hd).index_copy_(0, at[at >= 0], x[at >= 0])
        return got
    past, new = _lengths(case)
    out, at = torch.empty(s["rows"], H, hd, dtype=torch.float64, device=DEV), 0
    for i, (p, n) in enumerate(zip(past, new)):
        ids = s["table"][i, :_pages(p + n, case["page"])].long()
        k, v = (s[t][ids].reshape(-1, KV, hd)[:p + n].double() for t in ("k", "v"))
        q = s["q"][at:at + n].view(n, KV, H // KV, hd).double()
        hide = torch.triu(torch.ones(n, p + n, dtype=torch.bool, device=DEV), p + 1)
        for h in range(KV):
            a = (q[:, h].reshape(-1, hd) @ k[:, h].t().contiguous()).view(n, H // KV, p + n) / math.sqrt(hd)
            a = torch.softmax(a.masked_fill(hide[:, None], -math.inf), -1).view(-1, p + n)
            out[at:at + n, h * (H // KV):(h + 1) * (H // KV)] = (a @ v[:, h].contiguous()).view(n, H // KV, hd)
        at += n
    return out.view(s["rows"], H * hd)
