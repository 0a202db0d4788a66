"""The paged-cache operators against plain 64-bit restatements."""
import numpy as np
import pytest

import pitorch_amd as pa
from pitorch_amd._ffi import check
from tests import _paged as R

pytestmark = pytest.mark.gpu


def dev(a):
    from pitorch_amd._hip import DeviceArray
    return DeviceArray.from_host(np.ascontiguousarray(a))


def sync():
    check(pa.load_ptmi().ptmi_sync())


# ── plan ─────────────────────────────────────────────────────────────────

def run_plan(past, fresh, pool, n_pages, page, table, max_rows, alias=False):
    L = pa.load_ptmi()
    S, W = table.shape
    stack = np.full(n_pages + 1, -9, np.int32)
    stack[:len(pool)] = pool
    d = dict(past=dev(np.array(past + [0], np.int32)), fresh=dev(np.array(fresh + [0], np.int32)), pool=dev(stack),
             count=dev(np.array([len(pool)], np.int32)), table=dev(table.astype(np.int32).reshape(-1)))
    o = {n: dev(np.full(c + 1, -77, np.int32)) for n, c in
         dict(kv=S, left=1, start=S + 1, pos=max_rows, slot=max_rows, status=1).items()}
    if alias:
        o["kv"], o["left"] = d["past"], d["count"]
    check(L.ptmi_paged_plan_dev(d["past"].ptr, d["fresh"].ptr, S, d["pool"].ptr, d["count"].ptr, n_pages, page, d["table"].ptr, W,
                                o["kv"].ptr, o["left"].ptr, o["start"].ptr, o["pos"].ptr, o["slot"].ptr, max_rows, o["status"].ptr, None))
    sync()
    got = {n: a.download() for n, a in o.items()}
    if not alias:
        assert all(a[-1] == -77 for a in got.values())              # nothing past the ends
    got["pool"], got["table"] = d["pool"].download(), d["table"].download().reshape(S, W)
    assert got["pool"][-1] == -9
    return got


def check_plan(past, fresh, pool, n_pages, page, table, max_rows, alias=False):
    want_table = table.copy()
    kv, want_pool, start, pos, slot, status = R.plan(past, fresh, pool, n_pages, page, want_table, max_rows)
    g = run_plan(past, fresh, pool, n_pages, page, table, max_rows, alias)
    S = len(past)
    assert g["status"][0] == status
    assert g["kv"][:S].tolist() == kv.tolist() and g["start"][:S + 1].tolist() == start.tolist()
    assert g["pos"][:max_rows].tolist() == pos.tolist() and g["slot"][:max_rows].tolist() == slot.tolist()
    assert g["left"][0] == len(want_pool) and g["pool"][:len(want_pool)].tolist() == want_pool
    assert np.array_equal(g["table"], want_table)
    return status


def make_requests(rng, S, page, past_hi, new_hi, ended):
    past = [int(rng.integers(0, past_hi + 1)) for _ in range(S)]
    fresh = [-1 if rng.random() < ended else int(rng.integers(0, new_hi + 1)) for _ in range(S)]
    W = max(1, max(R.pages_for(p + max(f, 0), page) for p, f in zip(past, fresh)))
    used = sum(R.pages_for(p, page) for p in past)
    need = sum(R.pages_for(p + f, page) - R.pages_for(p, page) for p, f in zip(past, fresh) if f > 0)
    n_pages = used + need + 3
    ids = rng.permutation(n_pages)
    table, at = np.full((S, W), -1, np.int32), 0
    for i, p in enumerate(past):
        n = R.pages_for(p, page)
        table[i, :n] = ids[at:at + n]
        at += n
    return past, fresh, ids[at:].tolist(), n_pages, table, sum(max(f, 0) for f in fresh)


@pytest.mark.parametrize("S,page,past_hi,new_hi,ended", [
    (1, 16, 0, 1, 0), (1, 1, 5, 7, 0), (3, 16, 40, 1, 0.5), (64, 16, 1000, 1, 0.1), (5, 24, 300, 700, 0.2),
    (1024, 8, 60, 3, 0.2), (1025, 16, 90, 2, 0.1), (2500, 7, 30, 9, 0.3), (40, 64, 4000, 900, 0.1), (9, 128, 100, 100, 1.0)])
def test_plan(S, page, past_hi, new_hi, ended):
    rng = np.random.default_rng(S * 131 + page)
    past, fresh, pool, n_pages, table, rows = make_requests(rng, S, page, past_hi, new_hi, ended)
    assert check_plan(past, fresh, pool, n_pages, page, table, rows + int(rng.integers(0, 40))) == 0
    assert check_plan(past, fresh, pool, n_pages, page, table, rows, alias=True) == 0


def test_plan_many_rows():
    """More rows than one workgroup writes in a few turns, and requests of very different lengths."""
    past, fresh = [0, 5, 0, 33, 7], [0, 30000, 1, 0, 12345]
    page = 16
    need = sum(R.pages_for(p + f, page) for p, f in zip(past, fresh))
    ids = np.random.default_rng(5).permutation(need + 9)
    W = R.pages_for(30005, page)
    table, at = np.full((5, W), -1, np.int32), 0
    for i, p in enumerate(past):
        n = R.pages_for(p, page)
        table[i, :n] = ids[at:at + n]
        at += n
    assert check_plan(past, fresh, ids[at:].tolist(), need + 9, page, table, 45000) == 0
    assert check_plan(past, fresh, ids[at:].tolist(), need + 9, page, table, 45000, alias=True) == 0
    for alias in (False, True):                                # refused by all workgroups alike
        assert check_plan(past, fresh, ids[at:].tolist(), need + 9, page, table, 42000, alias) == 4
        assert check_plan(past, fresh, ids[at:-12].tolist(), need + 9, page, table, 45000, alias) == 1


@pytest.mark.parametrize("what", ["pool", "width", "rows", "past", "fresh", "overflow", "huge", "count", "back"])
def test_plan_refuses_as_a_whole(what):
    past, fresh, page, n_pages = [20, 3, 16], [5, -1, 20], 8, 20
    table = np.full((3, 6), -1, np.int32)
    table[0, :3], table[1, :1], table[2, :2] = (7, 2, 9), (4,), (0, 1)
    pool, max_rows = [11, 12, 13, 14], 30
    assert check_plan(past, fresh, pool, n_pages, page, table, max_rows) == 0
    if what == "pool":
        pool = [11, 12]
    elif what == "width":
        fresh[2] = 40
    elif what == "rows":
        max_rows = 24
    elif what == "past":
        past[0] = -1
    elif what == "fresh":
        fresh[0] = -2
    elif what == "overflow":
        past[0], fresh[0] = 2**31 - 2, 9
    elif what == "huge":                                     # sums past 32 bits
        fresh[:] = [2**31 - 100, 2**31 - 100, 2**31 - 100]
        past[:] = [0, 0, 0]
    elif what == "count":
        pool = list(range(20)) + [3]
    elif what == "back":                                     # more pages come back than there is room for
        pool = list(range(20))
    if what in ("count",):
        g = run_plan(past, fresh, pool[:20], n_pages, page, table, max_rows)
        assert g["status"][0] == 8
        return
    assert check_plan(past, fresh, pool, n_pages, page, table, max_rows) != 0


def test_plan_passes_on_bad_page_numbers():
    """Numbers outside the cache move as they are, and their positions have no slot."""
    table = np.full((3, 4), -1, np.int32)
    table[0, :3], table[1, :1], table[2, :2] = (7, 2**31 - 1, 9), (-5,), (20, 1)
    # the last request needs five pages of a table of four: refused for that, not for the numbers
    assert check_plan([17, 8, 16], [9, -1, 20], [11, 2**30, 13, -2**31], 20, 8, table, 40) == 2
    assert check_plan([17, 8, 16], [9, -1, 16], [11, 2**30, 13, -2**31], 20, 8, table, 40) == 0


def test_plan_of_most_requests():
    rng = np.random.default_rng(3)
    for S in (8192, 8191):
        past, fresh, pool, n_pages, table, rows = make_requests(rng, S, 16, 20, 2, 0.2)
        assert check_plan(past, fresh, pool, n_pages, 16, table, rows, alias=S == 8191) == 0


def test_plan_without_requests():
    g = run_plan([], [], [3, 1], 5, 16, np.zeros((0, 2), np.int32), 4)
    assert g["start"][0] == 0 and g["left"][0] == 2 and g["status"][0] == 0 and g["slot"][:4].tolist() == [-1] * 4


# ── store ────────────────────────────────────────────────────────────────

def rope_table(n, hd, rng):
    a = rng.uniform(-3, 3, (n, hd // 2))
    return np.stack((np.cos(a), np.sin(a)), -1).astype(np.float32)


LAYOUTS = {"tokens": lambda P, KV, hd: (P * KV * hd, KV * hd, hd),            # [page][position][head][hd]
           "heads": lambda P, KV, hd: (P * KV * hd, hd, P * hd),              # [page][head][position][hd]
           "padded": lambda P, KV, hd: (P * KV * (hd + 4) + 12, KV * (hd + 4), hd + 4)}


@pytest.mark.parametrize("rows,heads,kv,hd,page,kind,layout,with_rope,with_q", [
    (1, 6, 6, 48, 16, pa.F32, "tokens", 1, 1), (7, 12, 12, 64, 16, pa.F32, "heads", 1, 1), (33, 8, 2, 128, 24, pa.BF16, "tokens", 1, 1),
    (5, 3, 1, 36, 1, pa.BF16, "padded", 1, 1), (300, 4, 4, 4, 7, pa.F32, "padded", 0, 1), (19, 20, 4, 80, 64, pa.BF16, "heads", 1, 0),
    (64, 1, 1, 64, 16, pa.F32, "tokens", 0, 0), (66000, 1, 1, 4, 64, pa.F32, "tokens", 1, 1)])
@pytest.mark.parametrize("in_place", [False, True])
def test_store(rows, heads, kv, hd, page, kind, layout, with_rope, with_q, in_place):
    rng = np.random.default_rng(rows + hd)
    n_pages = R.pages_for(rows, page) + 2
    st = LAYOUTS[layout](page, kv, hd)
    size = n_pages * st[0] + 16
    ld, n_pos = (heads + 2 * kv) * hd + 8, 50
    x = rng.standard_normal((rows, ld)).astype(np.float32)
    slot = rng.permutation(n_pages * page)[:rows].astype(np.int32)
    pos = rng.integers(0, n_pos, rows).astype(np.int32)
    if rows > 4:
        slot[2], slot[rows - 1] = -1, n_pages * page          # skipped
        if with_rope:
            pos[3], pos[1] = -1, n_pos
    rope = rope_table(n_pos, hd, rng)
    dt = np.uint16 if kind == pa.BF16 else np.float32
    fill = rng.integers(0, 1000, size).astype(dt)
    dk, dv, dx = dev(fill), dev(fill), dev(x.reshape(-1))
    ldo = ld if in_place else heads * hd + 4
    q0 = np.full((rows, ldo), R.SENTINEL, np.float32)
    dq = dx if in_place else dev(q0.reshape(-1))
    dpos, dslot, drope = dev(pos), dev(slot), dev(rope.reshape(-1))
    c = R.pages_struct(dk.ptr, dv.ptr, kind, n_pages, page, kv, hd, st)
    check(pa.load_ptmi().ptmi_paged_store_dev(R.byref(c), dx.ptr if with_q else None, ld, dq.ptr if with_q else None, ldo, heads,
                                              dx.ptr + 4 * heads * hd, dx.ptr + 4 * (heads + kv) * hd, ld,
                                              dpos.ptr if with_rope else None, dslot.ptr, rows,
                                              drope.ptr if with_rope else None, n_pos if with_rope else 0, None))
    sync()
    live = (slot >= 0) & (slot < n_pages * page)
    if with_rope:
        live &= (pos >= 0) & (pos < n_pos)
    q, k, v = (t.reshape(rows, -1, hd) for t in np.split(x[:, :(heads + 2 * kv) * hd], [heads * hd, (heads + kv) * hd], 1))
    if with_rope:
        p = np.where(live, pos, 0)
        q, k = R.rotate(q, p, rope), R.rotate(k, p, rope)
    code = R.bf16 if kind == pa.BF16 else (lambda t: t)
    for d, t in ((dk, k), (dv, v)):
        want = fill.copy()
        want[R.place(st, slot[live], page, kv, hd)] = code(t[live])
        assert np.array_equal(d.download().view(np.uint8), want.view(np.uint8))      # every bit, also between the rows
    got, want = dq.download().reshape(rows, ldo), (x if in_place else q0).copy()
    if with_q:
        want[live, :heads * hd] = q[live].reshape(-1, heads * hd)
    assert np.array_equal(got, want)


def test_store_rounds_to_nearest_even():
    x = np.array([1.0, 1.00390625, 1.01171875, -1.00390625, 1.0039063, np.inf, -np.inf, np.nan, 3.3961776e38, 1e-40, -0.0, 65535.0], np.float32)
    dk, dv = dev(np.zeros(64, np.uint16)), dev(np.zeros(64, np.uint16))
    dx, ds = dev(x), dev(np.array([1], np.int32))
    c = R.pages_struct(dk.ptr, dv.ptr, pa.BF16, 1, 4, 1, 12)
    check(pa.load_ptmi().ptmi_paged_store_dev(R.byref(c), None, 12, None, 12, 1, dx.ptr, dx.ptr, 12, None, ds.ptr, 1, None, 0, None))
    sync()
    got = dk.download()[12:24]
    assert got.tolist() == R.bf16(x).tolist()
    assert got.tolist()[:4] == [0x3F80, 0x3F80, 0x3F82, 0xBF80] and got[8] == 0x7F80


# ── attention ────────────────────────────────────────────────────────────

def run_attention(reqs, heads, kv, hd, page, kind, layout="tokens", seed=0, max_new=None, scale=None, extra_rows=0, q_scale=1.5,
                  edit=None, stream=None, first_row=0, stale=np.nan, repeat=1):
    """reqs: (cached tokens before the step, new tokens) per request.  Positions that no row may see hold `stale`."""
    rng = np.random.default_rng(seed)
    L = pa.load_ptmi()
    S = len(reqs)
    lens = [p + n for p, n in reqs]
    W = max(1, max(R.pages_for(t, page) for t in lens))
    n_pages = sum(R.pages_for(t, page) for t in lens) + 2
    ids = rng.permutation(n_pages)
    table, at = np.full((S, W), 2**30, np.int32), 0
    k = np.full((n_pages * page, kv, hd), stale, np.float32)
    v = np.full((n_pages * page, kv, hd), stale, np.float32)
    for i, t in enumerate(lens):
        n = R.pages_for(t, page)
        table[i, :n] = ids[at:at + n]
        at += n
        tok = np.arange(t)
        slots = table[i, tok // page].astype(np.int64) * page + tok % page
        k[slots], v[slots] = (rng.standard_normal((t, kv, hd)).astype(np.float32) for _ in range(2))
    start = (np.concatenate(([0], np.cumsum([n for _, n in reqs]))) + first_row).astype(np.int32)
    kv_len = np.array(lens, np.int32)
    rows = int(start[-1]) + extra_rows
    q = (rng.standard_normal((rows, heads, hd)) * q_scale).astype(np.float32)
    scale = hd ** -0.5 if scale is None else scale
    d = dict(k=k, v=v, table=table, start=start, kv_len=kv_len, q=q)
    if edit:
        edit(d)
    st = LAYOUTS[layout](page, kv, hd)
    size = n_pages * st[0] + 16
    code = R.bf16 if kind == pa.BF16 else (lambda t: t)
    slots = np.arange(n_pages * page)
    mem = []
    for t in (d["k"], d["v"]):
        m = np.full(size, 0x7FC1 if kind == pa.BF16 else np.nan, np.uint16 if kind == pa.BF16 else np.float32)
        m[R.place(st, slots, page, kv, hd)] = code(t)
        mem.append(dev(m))
    if kind == pa.BF16:
        d["k"], d["v"] = R.from_bf16(R.bf16(d["k"])), R.from_bf16(R.bf16(d["v"]))
    ldq, ldo = heads * hd + 4, heads * hd + 8
    qm = np.full((max(rows, 1), ldq), np.nan, np.float32)
    qm[:rows, :heads * hd] = d["q"].reshape(rows, -1)
    om = np.full((max(rows, 1), ldo), R.SENTINEL, np.float32)
    dq, do = dev(qm.reshape(-1)), dev(om.reshape(-1))
    dt, ds, dl = dev(d["table"].reshape(-1)), dev(d["start"]), dev(d["kv_len"])
    c = R.pages_struct(mem[0].ptr, mem[1].ptr, kind, n_pages, page, kv, hd, st)
    top = max([n for _, n in reqs] + [0]) if max_new is None else max_new
    nb = L.ptmi_paged_attention_work(R.byref(c), heads, top)
    assert nb > 0
    dw = dev(np.full((nb + 3) // 4 + 8, np.nan, np.float32))      # whatever it holds
    for _ in range(repeat):
        check(L.ptmi_paged_attention_dev(R.byref(c), dt.ptr, W, ds.ptr, dl.ptr, S, top, dq.ptr, ldq, do.ptr, ldo, rows, heads, scale,
                                         dw.ptr, nb, stream))
    sync()
    assert np.isnan(dw.download()[(nb + 3) // 4:]).all()
    got = do.download().reshape(-1, ldo)
    assert (got[:, heads * hd:] == R.SENTINEL).all()
    got = got[:rows, :heads * hd].reshape(rows, heads, hd)
    want = np.full((rows, heads, hd), np.float64(R.SENTINEL))
    bound = R.attention(d["q"], d["k"], d["v"], d["table"].astype(np.int64), page, n_pages, d["start"], d["kv_len"], scale, want)
    return got, want, bound


def assert_close(got, want, bound):
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (np.argwhere(bad)[:5].tolist(), got[bad][:3], want[bad][:3], bound[bad][:3], bad.sum())


CASES = [
    # one token each: the shortest lengths, page borders
    ([(0, 1)], 6, 6, 48, 16, pa.F32, "tokens"),
    ([(0, 1), (15, 1), (16, 1), (17, 1), (63, 1), (64, 1), (200, 1)], 12, 12, 64, 16, pa.F32, "heads"),
    ([(1, 1), (300, 1), (31, 1)], 4, 2, 36, 24, pa.F32, "padded"),
    ([(100, 1), (999, 1)], 8, 1, 128, 64, pa.BF16, "tokens"),
    ([(77, 1)], 32, 2, 80, 7, pa.BF16, "heads"),
    ([(50, 1), (3, 1)], 40, 2, 64, 16, pa.F32, "tokens"),          # 20 heads share one
    ([(130, 1)], 3, 1, 4, 1, pa.F32, "tokens"),
    ([(40, 1)], 2, 2, 12, 3, pa.BF16, "padded"),
    ([(2100, 1)], 2, 2, 64, 16, pa.F32, "tokens"),
    # two to four rows a key head: two and three tokens, heads that share
    ([(0, 2), (62, 2), (129, 1), (40, 0)], 3, 3, 64, 16, pa.F32, "tokens"),
    ([(0, 3), (500, 3), (13, 2)], 2, 2, 48, 20, pa.F32, "heads"),
    ([(33, 2), (0, 1), (700, 2)], 4, 2, 128, 32, pa.BF16, "tokens"),
    ([(33, 4), (90, 1)], 2, 2, 100, 6, pa.BF16, "padded"),
    ([(65, 1), (70, 1)], 6, 2, 96, 16, pa.BF16, "heads"),
    ([(65, 4), (70, 3)], 1, 1, 128, 16, pa.F32, "tokens"),
    # a few tokens
    ([(0, 2), (5, 3), (100, 8), (30, 0), (7, 1)], 6, 6, 48, 16, pa.F32, "tokens"),
    ([(700, 4), (0, 5)], 8, 2, 64, 16, pa.BF16, "tokens"),
    # chunks
    ([(0, 64)], 2, 2, 64, 16, pa.F32, "tokens"),
    ([(0, 130), (65, 33), (200, 17)], 2, 2, 64, 16, pa.F32, "heads"),
    ([(37, 100), (0, 1), (500, 1), (3, 0), (0, 129)], 4, 2, 48, 24, pa.F32, "padded"),
    ([(300, 70)], 6, 2, 128, 100, pa.BF16, "tokens"),
    ([(10, 90), (0, 19)], 5, 1, 80, 24, pa.BF16, "heads"),
    ([(0, 200)], 1, 1, 36, 8, pa.F32, "tokens"),
    ([(12, 40)], 1, 1, 4, 5, pa.BF16, "tokens"),
    ([(60, 50)], 3, 3, 100, 16, pa.F32, "tokens"),
    ([(60, 33)], 20, 1, 64, 16, pa.F32, "tokens"),
    ([(1000, 128)], 1, 1, 96, 32, pa.F32, "tokens"),
    ([(0, 300), (513, 257)], 1, 1, 128, 16, pa.F32, "tokens"),
    ([(5, 9000)], 1, 1, 4, 64, pa.F32, "tokens"),                  # more than 64 tiles of rows
    ([(100, 3), (7, 64)], 128, 1, 4, 16, pa.F32, "tokens"),        # the most heads that share one
]


@pytest.mark.parametrize("reqs,heads,kv,hd,page,kind,layout", CASES)
def test_attention(reqs, heads, kv, hd, page, kind, layout):
    assert_close(*run_attention(reqs, heads, kv, hd, page, kind, layout, seed=hd + len(reqs)))


@pytest.mark.parametrize("case", [2, 16, 19])
def test_attention_without_a_bound_on_rows(case):
    """max_new 0 (not known), rows before, behind and outside the requests left as they were, a second call over the same work."""
    reqs, heads, kv, hd, page, kind, layout = CASES[case]
    assert_close(*run_attention(reqs, heads, kv, hd, page, kind, layout, seed=9, max_new=0, extra_rows=5, first_row=3, repeat=2))


@pytest.mark.parametrize("kind", [pa.F32, pa.BF16])
@pytest.mark.parametrize("new", [1, 3, 80])
def test_attention_rows_that_see_nothing(kind, new):
    """Lengths shorter than the new rows, negative lengths, pages outside the cache, whole and in the middle."""
    def edit(d):
        d["kv_len"][0] = new // 2                            # the first rows stand before position 0
        d["kv_len"][1] = 0
        d["kv_len"][2] = -5
        d["table"][3, :] = -1
        d["table"][4, 1] = 2**31 - 1
        d["table"][4, 3] = -2**31
        d["kv_len"][5] = 2**31 - 1                           # longer than the table is wide: all the table holds
        d["table"][5, d["table"][5] == 2**30] = -1
    reqs = [(40, new), (40, new), (40, new), (40, new), (90, new), (30, new)]
    got, want, bound = run_attention(reqs, 4, 2, 64, 16, kind, seed=3, edit=edit, stale=0.0)
    assert_close(got, want, bound)
    assert (got[new:4 * new] == 0).all()


@pytest.mark.parametrize("new", [1, 70])
@pytest.mark.parametrize("scale", [0.0, -0.3, 3.0])
def test_attention_scales(new, scale):
    """No scale, a negative one, one that makes the softmax nearly a choice."""
    assert_close(*run_attention([(150, new), (9, new)], 2, 2, 64, 16, pa.F32, seed=4, scale=scale))


@pytest.mark.parametrize("new", [1, 8, 70])
@pytest.mark.parametrize("kind", [pa.F32, pa.BF16])
def test_attention_of_large_and_small_values(new, kind):
    """Keys and values of very different sizes from tile to tile and within a row."""
    def edit(d):
        rng = np.random.default_rng(1)
        n = len(d["k"])
        f = np.exp2(rng.integers(-30, 30, (n, 1, 1))).astype(np.float32)
        d["v"] *= f
        g = np.exp2(rng.integers(-8, 8, (1, 1, d["k"].shape[2]))).astype(np.float32)
        d["k"] *= g
        d["q"] /= g[0]
        d["v"][::7] = 0
    assert_close(*run_attention([(400, new), (33, new)], 2, 2, 64, 16, kind, seed=6, edit=edit, stale=1e30))


@pytest.mark.parametrize("new", [1, 70])
@pytest.mark.parametrize("what", ["k", "v", "q"])
@pytest.mark.parametrize("bad", [np.inf, np.nan])
def test_attention_of_values_that_are_not_finite(new, what, bad):
    """They reach the rows that see them, of their head, and no others."""
    base, _, _ = run_attention([(100, new), (50, new)], 2, 2, 64, 16, pa.F32, seed=8)
    hit = 20

    q_sign = np.zeros(2 * new)

    def edit(d):
        q_sign[:] = d["q"][:, 1, 5]
        if what == "q":
            d["q"][new, 1, 5] = bad
        else:
            d[what][d["table"][1, hit // 16] * 16 + hit % 16, 1, 5] = bad
    got, _, _ = run_attention([(100, new), (50, new)], 2, 2, 64, 16, pa.F32, seed=8, edit=edit)
    assert np.array_equal(got[:new], base[:new]) and np.array_equal(got[new:, 0], base[new:, 0])
    if what == "q":
        assert np.isnan(got[new, 1]).all() and np.isfinite(got[new + 1:]).all()
    elif what == "k":                                        # (an infinite key may have a score of -infinity)
        assert np.isnan(got[new:, 1][q_sign[new:] > 0 if bad == np.inf else slice(None)]).all()
    else:
        assert not np.isfinite(got[new:, 1, 5]).any() and np.isfinite(np.delete(got[new:, 1], 5, 1)).all()


@pytest.mark.parametrize("new", [2, 3, 8, 70])
@pytest.mark.parametrize("kind", [pa.F32, pa.BF16])
@pytest.mark.parametrize("what", ["k", "v"])
@pytest.mark.parametrize("bad", [np.inf, np.nan])
def test_attention_of_new_tokens_that_are_not_finite(new, kind, what, bad):
    """A new token's key or value reaches the rows from its own on, none before it."""
    at = 2 * new // 3                                         # the new token
    reqs = [(37, new), (20, new)]
    base, _, _ = run_attention(reqs, 2, 2, 64, 16, kind, seed=8)
    q = np.zeros(2 * new)

    def edit(d):
        q[:] = d["q"][:, 1, 5]
        pos = 37 + at
        d[what][d["table"][0, pos // 16] * 16 + pos % 16, 1, 5] = bad
    got, _, _ = run_attention(reqs, 2, 2, 64, 16, kind, seed=8, edit=edit)
    # (the scale of the tile's keys may have moved with them: a rounding, not the bits)
    assert np.isfinite(got[:at]).all() and np.allclose(got[:at], base[:at], rtol=0, atol=2e-5)
    assert np.allclose(got[:, 0], base[:, 0], rtol=0, atol=2e-5) and np.allclose(got[new:], base[new:], rtol=0, atol=2e-5)
    if what == "v":
        assert not np.isfinite(got[at:new, 1, 5]).any()
        rest = [i for i in range(64) if i != 5]
        assert np.allclose(got[at:new, 1][:, rest], base[at:new, 1][:, rest], rtol=0, atol=2e-5)
    else:
        seen = q[at:new] > 0 if bad == np.inf else slice(None)
        assert np.isnan(got[at:new, 1][seen]).all()


@pytest.mark.parametrize("news", [(0, 1), (0, 1, 2), (1, 3, 9), (0, 1, 25)])
def test_attention_of_many_requests(news):
    """More requests than a workgroup looks at in one turn."""
    rng = np.random.default_rng(len(news) + news[-1])
    reqs = [(int(rng.integers(0, 40)), int(rng.choice(news))) for _ in range(600)]
    assert_close(*run_attention(reqs, 2, 1, 32, 8, pa.F32, seed=12))
    assert_close(*run_attention(reqs, 1, 1, 16, 8, pa.BF16, seed=13, max_new=0))


@pytest.mark.parametrize("heads,new", [(5, 1), (8, 1), (16, 1), (1, 5), (2, 7), (1, 16)])
@pytest.mark.parametrize("hd", [4, 28, 64, 80, 96, 124, 128])
def test_attention_of_five_to_sixteen_rows(hd, heads, new):
    """Lengths around the pairs of 64 keys that such rows take at once, in both types of pages."""
    lens = [0, 1, 47, 62, 63, 64, 65, 111, 126, 127, 128, 129, 191, 200, 640]
    layout = ("tokens", "heads", "padded")[(hd + heads) % 3]
    page = (16, 7, 24)[new % 3]
    for kind in (pa.BF16, pa.F32):
        assert_close(*run_attention([(n, new) for n in lens], 2 * heads, 2, hd, page, kind, layout, seed=hd + new))


@pytest.mark.parametrize("new", [1, 2, 8, 70])
@pytest.mark.parametrize("kind", [pa.F32, pa.BF16])
@pytest.mark.parametrize("size", [1e-37, 1e-20, 1e37])
def test_attention_of_keys_and_queries_of_any_size(new, kind, size):
    """Queries that make up for the size of the keys; values at both ends of the type."""
    def edit(d):
        d["k"] *= np.float32(size)
        d["q"] *= np.float32(1 / size)
        d["v"] *= np.float32(1e36)
    assert_close(*run_attention([(100, new), (9, new)], 2, 2, 64, 16, kind, seed=21, edit=edit, stale=0.0))


@pytest.mark.parametrize("new", [1, 2, 40])
def test_attention_repeats_itself(new):
    """The same bits every time, in any company."""
    a = run_attention([(900, new)], 4, 2, 64, 16, pa.F32, seed=11)[0]
    b = run_attention([(900, new)], 4, 2, 64, 16, pa.F32, seed=11, repeat=3)[0]
    assert np.array_equal(a, b)


def test_attention_far_into_a_large_cache():
    """Element offsets past 32 bits: the pages lie more than 2^31 elements apart."""
    from pitorch_amd._hip import DeviceArray
    L = pa.load_ptmi()
    page, hd, heads, n_pages = 16, 64, 2, 3
    stride = 1100000000                                      # elements from page to page
    n = (n_pages - 1) * stride + page * heads * hd
    k, v = DeviceArray(n, np.uint16), DeviceArray(n, np.uint16)
    rng = np.random.default_rng(2)
    kk, vv = (rng.standard_normal((n_pages * page, heads, hd)).astype(np.float32) for _ in range(2))
    x = np.concatenate((kk, vv), 1).reshape(n_pages * page, -1)
    c = R.pages_struct(k.ptr, v.ptr, pa.BF16, n_pages, page, heads, hd, (stride, heads * hd, hd))
    dx, ds = dev(x.reshape(-1)), dev(np.arange(n_pages * page, dtype=np.int32))
    check(L.ptmi_paged_store_dev(R.byref(c), None, 0, None, 0, 1, dx.ptr, dx.ptr + 4 * heads * hd, 2 * heads * hd, None, ds.ptr,
                                 n_pages * page, None, 0, None))
    table, start, kv_len = np.array([[2, 0, 1]], np.int32), np.array([0, 30], np.int32), np.array([48], np.int32)
    q = rng.standard_normal((30, heads, hd)).astype(np.float32)
    for rows in (1, 30):
        start[1] = rows
        dq, do = dev(q.reshape(-1)), dev(np.zeros(q.size, np.float32))
        nb = L.ptmi_paged_attention_work(R.byref(c), heads, rows)
        dw = DeviceArray(nb, np.uint8)
        dt, dst, dl = dev(table.reshape(-1)), dev(start), dev(kv_len)
        check(L.ptmi_paged_attention_dev(R.byref(c), dt.ptr, 3, dst.ptr, dl.ptr, 1, rows, dq.ptr, heads * hd, do.ptr, heads * hd, rows,
                                         heads, 0.125, dw.ptr, nb, None))
        sync()
        want = np.zeros((rows, heads, hd))
        bound = R.attention(q[:rows], R.from_bf16(R.bf16(kk)), R.from_bf16(R.bf16(vv)), table.astype(np.int64), page, n_pages, start,
                            kv_len, 0.125, want)
        assert_close(do.download().reshape(30, heads, hd)[:rows], want, bound)
    k.free()
    v.free()
