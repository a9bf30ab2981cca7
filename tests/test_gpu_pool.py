"""The serving operators over a caller-owned page pool on the device, against plain forms in 64 bits: the plan, the
store, the attention and a run of them together, eager and as a captured graph."""
import itertools

import numpy as np
import pytest

import pool_oracle as po

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be(kg):
    b = kg.CudaBackend(kg.micro_config())
    yield b
    b.pool_status()
    b.close()


def _t(x, dtype=None):
    import torch
    return torch.as_tensor(np.asarray(x), dtype=dtype or torch.int32).cuda().contiguous()


# ---------------------------------------------------------------- plan

def _run_plan(be, page, n_pages, cached, new, table, free, n_free, max_tokens, in_place=False, stream=None):
    import torch
    n = len(cached)
    t, left = _t(table), _t([n_free])
    out = left if in_place else _t([12345])
    got = [torch.full((k,), 777, dtype=torch.int32, device="cuda") for k in (n + 2, n + 1, max_tokens + 1, max_tokens + 1, max_tokens + 1, 2)]
    c, a, f = _t(cached), _t(new), _t(free if len(free) else [0])
    be.pool_plan_dev(page, n_pages, n, c.data_ptr(), a.data_ptr(), t.data_ptr(), table.shape[1], f.data_ptr(), left.data_ptr(),
                     out.data_ptr(), max_tokens, *(x.data_ptr() for x in got), stream)
    torch.cuda.synchronize()
    assert all(int(x[-1]) == 777 for x in got)  # one past each output
    cu, kv, slots, req, pos, status = (x[:-1].cpu().numpy() for x in got)
    return int(status[0]), t.cpu().numpy(), int(out[0]), cu, kv, slots, req, pos


def _state(rng, page, n, old_hi, new_hi, spare=0, shrink=0):
    cached = rng.integers(0, old_hi + 1, n)
    new = rng.integers(0, new_hi + 1, n)
    if n > 2:
        cached[1], new[2] = 0, 0
    has, need = -(-cached // page), -(-(cached + new) // page)
    n_pages = int(need.sum()) + spare + 1
    perm = rng.permutation(n_pages)
    width = int(need.max(initial=0)) + 2
    table = np.full((n, width), -7)
    at = 0
    for r in range(n):
        table[r, : has[r]] = perm[at:at + has[r]]
        at += has[r]
    free = perm[at:]
    return cached, new, table, free, len(free) - shrink, n_pages


@pytest.mark.parametrize("page,n,old_hi,new_hi,pad,in_place", [
    (16, 1, 0, 1, 0, False), (16, 1, 40, 1, 3, True), (16, 3, 17, 5, 0, True), (32, 64, 1200, 1, 0, False),
    (64, 33, 500, 300, 100, True), (128, 700, 900, 40, 1, False), (16, 1024, 100, 1, 0, True), (16, 1025, 64, 33, 9, True),
    (16, 16384, 20, 3, 5, True), (16, 5, 100, 9000, 0, False), (16, 2, 3, 70000, 11, True),
])
def test_plan(be, page, n, old_hi, new_hi, pad, in_place):
    rng = np.random.default_rng(n * 1000 + new_hi)
    cached, new, table, free, n_free, n_pages = _state(rng, page, n, old_hi, new_hi, spare=rng.integers(0, 30))
    m = int(new.sum()) + pad
    want = po.plan(page, n_pages, cached, new, table, free, n_free, m)
    got = _run_plan(be, page, n_pages, cached, new, table, free, n_free, m, in_place)
    assert want[0] == 0
    for w, g in zip(want, got):
        np.testing.assert_array_equal(g, w)


@pytest.mark.parametrize("what", ["pages", "tokens", "width", "negative", "negative new", "n_free", "n_free below", "free entry",
                                  "last page", "overflow"])
def test_plan_that_does_not_fit_takes_nothing(be, what):
    rng = np.random.default_rng(5)
    cached, new, table, free, n_free, n_pages = _state(rng, 16, 40, 100, 50)
    cached[7], new[7] = 21, 9
    m = int(new.sum()) + 4
    table[7, 0], table[7, 1] = 0, 1
    if what == "pages":
        grow = int((-(-(cached + new) // 16) - -(-cached // 16)).sum())
        n_free = grow - 1
    elif what == "tokens":
        m = int(new.sum()) - 1
    elif what == "width":
        table = table[:, :-4].copy()
        cached[11], new[11] = 16 * table.shape[1], 1
    elif what == "negative":
        cached[3] = -1
    elif what == "negative new":
        new[3] = -2
    elif what == "n_free":
        n_free = n_pages + 1
    elif what == "n_free below":
        n_free = -1
    elif what == "free entry":
        free[n_free - 2] = n_pages
    elif what == "last page":
        table[7, 1] = -1
    elif what == "overflow":
        cached[3], new[3] = 2**31 - 1, 1
    free = np.concatenate([free, np.zeros(4, int)])  # n_free may point one past what was given
    want = po.plan(16, n_pages, cached, new, table, free, n_free, m)
    got = _run_plan(be, 16, n_pages, cached, new, table, free, n_free, m, in_place=True)
    assert want[0] == (-2 if what == "pages" else -1)
    for w, g in zip(want, got):
        np.testing.assert_array_equal(g, w)


def test_plan_of_nothing(be):
    got = _run_plan(be, 16, 4, [], [], np.zeros((0, 1), int), [1, 2], 2, 3)
    assert got[0] == 0 and got[2] == 2 and list(got[3]) == [0] and list(got[5]) == [-1] * 3
    got = _run_plan(be, 16, 4, [5], [0], np.full((1, 1), 2), [], 0, 0)
    assert got[0] == 0 and got[2] == 0 and list(got[4]) == [5]


# ---------------------------------------------------------------- store

LAYOUTS = ["page", "heads first", "apart"]


def _make_pool(kg, layout, n_pages, page, n_kv, d, dt):
    """(views [n_pages][page][n_kv][d] of K and V, the kg_pool), all NaN."""
    import torch
    td = {"bf16": torch.bfloat16, "f16": torch.float16}[dt]
    new = lambda *s: torch.full(s, float("nan"), dtype=td, device="cuda")  # noqa: E731
    if layout == "page":  # the framework's pages: K rows, then V rows
        m = new(n_pages, 2, page, n_kv, d)
        k, v = m[:, 0], m[:, 1]
    elif layout == "heads first":  # a head's rows together, pages of K and V alternating
        m = new(n_pages, 2, n_kv, page, d)
        k, v = m[:, 0].transpose(1, 2), m[:, 1].transpose(1, 2)
    else:  # two pools whose rows have room behind them
        k, v = new(n_pages, page, n_kv, d + 8)[..., :d], new(n_pages, page, n_kv, d + 8)[..., :d]
    assert k.stride() == v.stride()
    return k, v, kg.page_pool(k.data_ptr(), v.data_ptr(), n_pages, page, n_kv, d, dt, page_stride=k.stride(0),
                              row_stride=k.stride(1), head_stride=k.stride(2))


@pytest.mark.parametrize("src,dt,layout", list(itertools.product(["f32", "bf16", "f16"], ["bf16", "f16"], LAYOUTS)))
def test_store(kg, be, src, dt, layout):
    import torch
    page, n_kv, d, rows = (16, 3, 64, 37) if layout != "apart" else (32, 2, 128, 1)
    k, v, pool = _make_pool(kg, layout, 9, page, n_kv, d, dt)
    ts = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[src]
    g = torch.Generator(device="cuda").manual_seed(3)
    qkv = torch.randn(rows, 3, n_kv, d + 8, generator=g, device="cuda").to(ts)
    if rows > 1:
        qkv[1, 1, 0, :4] = torch.tensor([float("inf"), -float("inf"), float("nan"), 0.0])
    slots = torch.randperm(9 * page, generator=g, device="cuda")[:rows].to(torch.int32)
    if rows > 1:
        slots[5], slots[6], slots[7] = -1, -2**31, 9 * page  # two paddings and one past the pool
    kr, vr = qkv[:, 1, :, :d], qkv[:, 2, :, :d]
    be.pool_store_dev(pool, rows, slots.data_ptr(), src, kr.data_ptr(), vr.data_ptr(), kr.stride(0), kr.stride(1))
    torch.cuda.synchronize()
    for got, rows_ in ((k, kr), (v, vr)):
        want = torch.full((9 * page, n_kv, d), float("nan"), dtype=got.dtype, device="cuda")
        ok = (slots >= 0) & (slots < 9 * page)
        want[slots[ok].long()] = rows_[ok].to(got.dtype)  # one rounding, to the nearest even
        assert torch.equal(torch.nan_to_num(got.reshape(9 * page, n_kv, d).float(), 1e30, 2e30, -2e30),
                           torch.nan_to_num(want.float(), 1e30, 2e30, -2e30))
    if rows > 1:
        with pytest.raises(kg.KgError, match="rejected"):
            be.pool_status()
    be.pool_status()


# ---------------------------------------------------------------- attend

def _attend_case(kg, be, reqs, n_head, n_kv, d, page, dt, causal, layout="page", pad=0, seed=0, spread=1.0, stream=None, strided=False,
                 extra=1):
    """Runs one batch over pages that are NaN wherever nothing was stored, and checks every row."""
    import torch
    rng = np.random.default_rng(seed)
    td = {"bf16": torch.bfloat16, "f16": torch.float16}[dt]
    q_len, kv = [r[0] for r in reqs], [r[1] for r in reqs]
    need = [-(-x // page) for x in kv]
    n_pages = sum(need) + extra
    k, v, pool = _make_pool(kg, layout, n_pages, page, n_kv, d, dt)
    width = max(max(need, default=0), 1) + 1
    table = np.full((len(reqs), width), -3)
    perm = rng.permutation(n_pages)
    ks, vs, at = [], [], 0
    for r in range(len(reqs)):
        table[r, : need[r]] = perm[at:at + need[r]]
        kk, vv = (torch.from_numpy(rng.standard_normal((kv[r], n_kv, d))).mul(spread).to(td) for _ in range(2))
        for j in range(need[r]):
            m = min(page, kv[r] - j * page)
            k[int(table[r, j]), :m] = kk[j * page:j * page + m].cuda()
            v[int(table[r, j]), :m] = vv[j * page:j * page + m].cuda()
        ks.append(kk.double().numpy())
        vs.append(vv.double().numpy())
        at += need[r]
    cu = np.concatenate([[0], np.cumsum(q_len)]).astype(int)
    total = int(cu[-1]) + pad
    q = torch.from_numpy(rng.standard_normal((total, n_head, d))).mul(spread).to(td)
    scale = d ** -0.5
    if strided == "heads first":
        qd, out = q.transpose(0, 1).contiguous().cuda().transpose(0, 1), torch.full((total, n_head, d), 7.0, dtype=td, device="cuda")
    elif strided:  # q inside a fused projection's rows, out with heads first
        big = torch.zeros(total, n_head + 2 * n_kv, d, dtype=td)
        big[:, :n_head] = q
        qd = big.cuda()[:, :n_head]
        out = torch.full((n_head, total, d + 8), 7.0, dtype=td, device="cuda")[..., :d].transpose(0, 1)
    else:
        qd, out = q.cuda(), torch.full((total, n_head, d), 7.0, dtype=td, device="cuda")
    ws = torch.full((be.pool_attend_bytes(pool, len(reqs), n_head, total),), 0xFF, dtype=torch.uint8, device="cuda")  # NaN patterns
    cud, kvd, td_ = _t(cu), _t(kv if kv else [0]), _t(table if len(reqs) else [[0]])
    be.pool_attend_dev(pool, len(reqs), n_head, total, cud.data_ptr(), kvd.data_ptr(), td_.data_ptr(), width, qd.data_ptr(), qd.stride(0),
                       qd.stride(1), out.data_ptr(), out.stride(0), out.stride(1), scale, causal, ws.data_ptr(), ws.numel(), stream)
    torch.cuda.synchronize()
    be.pool_status()
    got = out.double().cpu().numpy()
    want, mine, mag, sco = po.attend(q.double().numpy(), ks, vs, cu, kv, scale, causal)
    np.testing.assert_array_equal(got[~mine], 7.0)
    # one rounding of the result, one of every probability to the pool's type (each half a step), f32 scores: a dot
    # product of d terms is off by at most d * 2^-24 of its absolute terms, which moves a probability by that much
    # relative to itself (once in the weights, once in their sum); exp and the running sums: 2^-18 for all the rest
    half = torch.finfo(td).eps / 2
    tol = half * np.abs(want) * 1.01 + mag * (half * 1.01 + 2 * d * 2.0 ** -24 * sco[..., None] + 2.0 ** -18)
    err = np.abs(got - want) - tol
    assert not np.isnan(got[mine]).any()
    assert (err[mine] <= 2.0 ** -24).all(), (err[mine].max(), np.unravel_index(err.argmax(), err.shape))
    return got


RAGGED = [(0, 0), (1, 1), (0, 40), (1, 17), (3, 2), (5, 0), (16, 16), (17, 33), (1, 700), (5, 400), (2, 128), (1, 129)]


@pytest.mark.parametrize("d,page,dt", list(itertools.product([64, 128], [16, 32, 64, 128], ["bf16", "f16"])))
def test_attend_ragged(kg, be, d, page, dt):
    _attend_case(kg, be, RAGGED, 4, 2, d, page, dt, 1, pad=3, seed=d + page)


@pytest.mark.parametrize("n_head,n_kv", [(1, 1), (3, 1), (12, 12), (10, 2), (7, 1), (32, 2), (64, 1), (24, 3)])
def test_attend_head_layouts(kg, be, n_head, n_kv):
    _attend_case(kg, be, [(1, 300), (9, 70), (1, 1), (40, 200)], n_head, n_kv, 64, 16, "bf16", 1, pad=1, seed=n_head)


@pytest.mark.parametrize("layout,strided,causal", list(itertools.product(LAYOUTS, [False, True, "heads first"], [0, 1])))
def test_attend_layouts_and_masks(kg, be, layout, strided, causal):
    _attend_case(kg, be, [(1, 90), (33, 50), (4, 3), (20, 260)], 6, 2, 128, 16, "bf16", causal, layout=layout, strided=strided, seed=9)


@pytest.mark.parametrize("reqs,n_head,n_kv,d,page", [
    ([(1, 5000)], 8, 1, 128, 16),           # one sequence: its positions split over the device
    ([(1, 4097), (1, 31), (1, 2048)], 4, 4, 64, 32),
    ([(130, 3000)], 8, 2, 128, 16),         # a chunk over a long prefix
    ([(300, 300), (1, 900), (257, 700)], 4, 4, 128, 16),
    ([(600, 600), (128, 128), (129, 1290)], 2, 1, 64, 64),
    ([(90, 1000), (43, 1000), (1, 77)], 6, 2, 128, 128),   # three rows a token
    ([(70, 333), (52, 52)], 10, 2, 64, 16),                # five
    ([(2, 900)] * 40, 4, 1, 128, 16),
    ([(20, 9000)], 8, 1, 128, 16),           # one tile's positions split over many CTAs
    ([(1, 70001), (1, 3)], 2, 1, 64, 128),
    ([(70, 70)], 1, 1, 64, 16),              # fewer rows than a tile of tokens
    ([(65, 200), (66, 65)], 2, 2, 128, 32),
    ([(2, 50), (3, 700), (9, 130)], 64, 1, 128, 16),
    ([(129, 20), (300, 150), (80, 0)], 2, 1, 128, 16),  # rows before position 0 in long requests
    ([(1, 130 + 3 * i) for i in range(200)], 4, 2, 64, 16),
])
def test_attend_long(kg, be, reqs, n_head, n_kv, d, page):
    for causal in (1, 0):
        _attend_case(kg, be, reqs, n_head, n_kv, d, page, "bf16", causal, seed=len(reqs))


@pytest.mark.parametrize("reqs", [[(1, 600)], [(200, 900)], [(6, 300), (1, 50)]])
def test_attend_peaked_scores(kg, be, reqs):
    # scores of some hundreds: one position takes nearly everything, running maxima jump
    _attend_case(kg, be, reqs, 4, 2, 128, 16, "bf16", 1, seed=4, spread=6.0)
    _attend_case(kg, be, reqs, 4, 2, 64, 16, "f16", 0, seed=5, spread=5.0)


def test_attend_repeats_bit_for_bit(kg, be):
    for reqs in ([(1, 3000), (1, 100)], [(300, 2000), (1, 800), (40, 40)]):
        a = _attend_case(kg, be, reqs, 8, 2, 128, 16, "bf16", 1, seed=3)
        b = _attend_case(kg, be, reqs, 8, 2, 128, 16, "bf16", 1, seed=3)
        np.testing.assert_array_equal(a, b)


def test_attend_far_pages(kg, be):
    """Element offsets past 2^31: pages at the end of a pool of 5 GB."""
    import torch
    page, n_kv, d = 16, 8, 128
    n_pages = 80000  # 16384 elements a page with K and V 32768: the last is at 2.6e9
    m = torch.empty(n_pages, 2, page, n_kv, d, dtype=torch.bfloat16, device="cuda")
    m[-4:] = torch.randn(4, 2, page, n_kv, d, device="cuda")
    pool = kg.page_pool(m.data_ptr(), m[0, 1].data_ptr(), n_pages, page, n_kv, d)
    for rows, kv in ((1, 60), (50, 60)):
        q = torch.randn(rows, 16, d, device="cuda").bfloat16()
        out = torch.zeros_like(q)
        ws = torch.empty(be.pool_attend_bytes(pool, 1, 16, rows), dtype=torch.uint8, device="cuda")
        table, cu, kvd = _t([[n_pages - 1, n_pages - 3, n_pages - 2, n_pages - 4]]), _t([0, rows]), _t([kv])
        be.pool_attend_dev(pool, 1, 16, rows, cu.data_ptr(), kvd.data_ptr(), table.data_ptr(), 4, q.data_ptr(), q.stride(0),
                           q.stride(1), out.data_ptr(), out.stride(0), out.stride(1), d ** -0.5, 1, ws.data_ptr(), ws.numel())
        be.pool_status()
        kk, vv = (m[table[0].long(), i].reshape(64, n_kv, d)[:kv].double().cpu().numpy() for i in (0, 1))
        want, _, mag, sco = po.attend(q.double().cpu().numpy(), [kk], [vv], [0, rows], [kv], d ** -0.5, 1)
        tol = 2.0 ** -8 * 1.01 * (np.abs(want) + mag) + mag * (2 * d * 2.0 ** -24 * sco[..., None] + 2.0 ** -18)
        assert (np.abs(out.double().cpu().numpy() - want) <= tol + 2.0 ** -24).all()


@pytest.mark.parametrize("rows", [1, 150])
def test_attend_reports_what_the_device_rejects(kg, be, rows):
    """Lengths that do not fit leave the rows alone; a table entry outside the pool reads as zeros."""
    import torch
    page, n_kv, d, h = 16, 2, 64, 4
    m = torch.randn(20, 2, page, n_kv, d, device="cuda").bfloat16()
    pool = kg.page_pool(m.data_ptr(), m[0, 1].data_ptr(), 20, page, n_kv, d)
    q = torch.randn(3 * rows, h, d, device="cuda").bfloat16()
    ws = torch.empty(be.pool_attend_bytes(pool, 3, h, 3 * rows), dtype=torch.uint8, device="cuda")
    table = torch.arange(30, device="cuda", dtype=torch.int32).view(3, 10) % 20

    def go(cu, kv, tab):
        out = torch.full_like(q, 7.0)
        cud, kvd, tabd = _t(cu), _t(kv), tab.contiguous()
        be.pool_attend_dev(pool, 3, h, 3 * rows, cud.data_ptr(), kvd.data_ptr(), tabd.data_ptr(), 10, q.data_ptr(), q.stride(0), q.stride(1),
                           out.data_ptr(), out.stride(0), out.stride(1), 0.125, 1, ws.data_ptr(), ws.numel())
        torch.cuda.synchronize()
        return out

    def near(out, r, kv, zero=()):  # request r's rows (the cut of its sums may differ with the others' lengths)
        kk, vv = (m[table[r].long(), i].reshape(160, n_kv, d).double().cpu().numpy()[:kv] for i in (0, 1))
        for z in zero:
            kk[z:z + page], vv[z:z + page] = 0, 0
        want, _, mag, sco = po.attend(q[r * rows:(r + 1) * rows].double().cpu().numpy(), [kk], [vv], [0, rows], [kv], 0.125, 1)
        tol = 2.0 ** -8 * 1.01 * (np.abs(want) + mag) + mag * (2 * d * 2.0 ** -24 * sco[..., None] + 2.0 ** -18)
        return (np.abs(out[r * rows:(r + 1) * rows].double().cpu().numpy() - want) <= tol + 2.0 ** -24).all()

    good = go([0, rows, 2 * rows, 3 * rows], [155, 160, 150], table)
    be.pool_status()
    assert near(good, 0, 155) and near(good, 1, 160) and near(good, 2, 150)
    for cu, kv in (([0, rows, 2 * rows, 3 * rows + 1], [155, 160, 150]), ([0, rows, 2 * rows, 3 * rows], [155, 160, 161]),
                   ([0, rows, 2 * rows, 3 * rows], [155, 160, -1]), ([0, rows, 2 * rows, rows - 1], [155, 160, 150])):
        out = go(cu, kv, table)
        assert near(out, 0, 155) and near(out, 1, 160) and (out[2 * rows:] == 7).all()
        with pytest.raises(kg.KgError, match="rejected"):
            be.pool_status()
    for bad in (-1, 20, 2**31 - 1, -2**31):
        tab = table.clone()
        tab[1, 3] = bad
        out = go([0, rows, 2 * rows, 3 * rows], [155, 160, 150], tab)
        assert torch.equal(out[:rows], good[:rows]) and torch.equal(out[2 * rows:], good[2 * rows:])
        with pytest.raises(kg.KgError, match="rejected"):
            be.pool_status()
        assert near(out, 1, 160, zero=[48])
    be.pool_status()


def test_attend_of_nothing(kg, be):
    _attend_case(kg, be, [(0, 0), (0, 30)], 4, 2, 64, 16, "bf16", 1, pad=4)
    _attend_case(kg, be, [(7, 0), (1, 0)], 4, 2, 64, 16, "bf16", 1, pad=4)
    _attend_case(kg, be, [(7, 0), (140, 0)], 4, 2, 64, 16, "bf16", 0)


def test_calls_on_two_streams(kg, be):
    """Calls that overlap on the device, on streams of their own with a workspace each, against each of them alone."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(7)
    page, n_kv, d, h = 16, 2, 128, 8
    m = torch.randn(400, 2, page, n_kv, d, generator=g, device="cuda").bfloat16()
    pool = kg.page_pool(m.data_ptr(), m[0, 1].data_ptr(), 400, page, n_kv, d)
    calls = []
    for q_len, kv in (([1, 1, 3], [3000, 100, 900]), ([200, 1], [900, 400]), ([40, 33], [40, 2000])):
        n, total = len(kv), sum(q_len)
        table = torch.randint(0, 400, (n, 200), generator=g, device="cuda", dtype=torch.int32)
        q = torch.randn(total, h, d, generator=g, device="cuda").bfloat16()
        cu, kvd = _t(np.concatenate([[0], np.cumsum(q_len)])), _t(kv)
        out = torch.zeros_like(q)
        ws = torch.empty(be.pool_attend_bytes(pool, n, h, total), dtype=torch.uint8, device="cuda")
        s = torch.cuda.Stream()

        def call(n=n, total=total, cu=cu, kvd=kvd, table=table, q=q, out=out, ws=ws, s=s):
            be.pool_attend_dev(pool, n, h, total, cu.data_ptr(), kvd.data_ptr(), table.data_ptr(), 200, q.data_ptr(), q.stride(0), q.stride(1),
                               out.data_ptr(), out.stride(0), out.stride(1), d ** -0.5, 1, ws.data_ptr(), ws.numel(), s.cuda_stream)
        torch.cuda.synchronize()
        call()
        torch.cuda.synchronize()
        calls.append((call, out, out.clone()))
    for _ in range(20):
        for call, out, _ in calls:
            call()
    torch.cuda.synchronize()
    be.pool_status()
    for _, out, alone in calls:
        assert torch.equal(out, alone)


# ---------------------------------------------------------------- together

class Server:
    """Requests over one pool, every step plan -> project -> store -> attend -> logits -> sample on the device. Buffers are
    fixed, so that a step can be captured; padding rows stand behind the last request's."""

    def __init__(self, kg, be, n_req, max_tokens, seed=0):
        import torch
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.be, self.n, self.m, self.page, self.h, self.n_kv, self.d, self.vocab = be, n_req, max_tokens, 16, 4, 2, 64, 211
        self.n_pages, self.width = 96, 12
        rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        self.emb, self.pos_emb = rnd(self.vocab, 128), rnd(self.width * self.page, 128)
        self.w = rnd(128, (self.h + 2 * self.n_kv) * self.d) * 128 ** -0.5
        self.head = (rnd(self.h * self.d, self.vocab) * 0.3)
        self.k, self.v, self.pool = _make_pool(kg, "page", self.n_pages, self.page, self.n_kv, self.d, "bf16")
        z = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
        self.cached, self.new, self.table = z(n_req), z(n_req), z(n_req, self.width) - 1
        self.free, self.n_free = torch.randperm(self.n_pages, generator=g, device="cuda").to(torch.int32), z(1) + self.n_pages
        self.cu, self.kv, self.slots, self.req, self.pos, self.status = z(n_req + 1), z(n_req), z(self.m), z(self.m), z(self.m), z(1)
        self.tokens, self.next = z(self.m), z(n_req)
        self.out = torch.zeros(self.m, self.h, self.d, dtype=torch.bfloat16, device="cuda")
        self.ws = torch.empty(be.pool_attend_bytes(self.pool, n_req, self.h, self.m), dtype=torch.uint8, device="cuda")
        self.u, self.top_p = torch.zeros(n_req, device="cuda"), torch.full((n_req,), 0.9, device="cuda")
        self.logits = torch.zeros(n_req, self.vocab, device="cuda")

    def step(self):
        import torch
        s, p = torch.cuda.current_stream().cuda_stream, lambda x: x.data_ptr()  # noqa: E731
        self.be.pool_plan_dev(self.page, self.n_pages, self.n, p(self.cached), p(self.new), p(self.table), self.width, p(self.free),
                              p(self.n_free), p(self.n_free), self.m, p(self.cu), p(self.kv), p(self.slots), p(self.req), p(self.pos),
                              p(self.status), s)
        x = self.emb[self.tokens.long()] + self.pos_emb[self.pos.long().clamp(min=0)]
        self.qkv = x @ self.w
        a, b = self.h * self.d, (self.h + self.n_kv) * self.d
        self.be.pool_store_dev(self.pool, self.m, p(self.slots), "f32", p(self.qkv) + a * 4, p(self.qkv) + b * 4, self.qkv.stride(0), self.d, s)
        self.q = self.qkv[:, :a].reshape(self.m, self.h, self.d).bfloat16()
        self.be.pool_attend_dev(self.pool, self.n, self.h, self.m, p(self.cu), p(self.kv), p(self.table), self.width, p(self.q), self.q.stride(0),
                                self.q.stride(1), p(self.out), self.out.stride(0), self.out.stride(1), self.d ** -0.5, 1, p(self.ws),
                                self.ws.numel(), s)
        last = (self.cu[1:] - 1).clamp(min=0).long()
        self.logits.copy_(self.out[last].reshape(self.n, -1).float() @ self.head)
        self.be.sample_logits_dev(self.n, self.vocab, "f32", p(self.logits), self.vocab, None, None, p(self.top_p), None, p(self.u), p(self.next), s)
        self.cached.copy_(self.kv)


@pytest.mark.parametrize("captured", [False, True])
def test_a_run_of_them(kg, be, captured):
    """Prompts of unlike lengths, then steps in which requests go on, rest or bring several tokens: every step's attention
    and tokens against histories kept apart from the pages, eager and replayed from one graph."""
    import torch
    rng = np.random.default_rng(1)
    n, m = 5, 96
    srv = Server(kg, be, n, m)
    side, graph = torch.cuda.Stream(), None
    hist_k = [np.zeros((0, srv.n_kv, srv.d)) for _ in range(n)]
    hist_v = [np.zeros((0, srv.n_kv, srv.d)) for _ in range(n)]
    plan = [[40, 1, 17, 0, 30], [1, 1, 1, 33, 1], [1, 1, 0, 1, 1], [1, 5, 1, 1, 0], [1, 1, 1, 1, 1], [0, 0, 0, 0, 0], [60, 1, 1, 1, 16]]
    nxt = rng.integers(0, srv.vocab, n)
    for t, new in enumerate(plan):
        toks = []
        for r, a in enumerate(new):
            toks += [int(nxt[r])] * (a == 1) if a <= 1 else [int(x) for x in rng.integers(0, srv.vocab, a)]
        before = srv.out.clone()
        srv.new.copy_(_t(new))
        srv.tokens.copy_(_t(toks + [0] * (m - len(toks))))
        u = rng.random(n).astype(np.float32)
        srv.u.copy_(torch.from_numpy(u).cuda())
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.default_stream())
            if not captured or t == 0:
                srv.step()
            else:
                if graph is None:
                    side.synchronize()
                    state = [x.clone() for x in (srv.n_free, srv.table, srv.cached)]
                    graph = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(graph, stream=side):
                        srv.step()
                    for x, y in zip((srv.n_free, srv.table, srv.cached), state):
                        x.copy_(y)
                graph.replay()
        side.synchronize()
        be.pool_status()
        assert int(srv.status) == 0
        total = sum(new)
        kk = srv.qkv[:total].bfloat16().double().cpu().numpy().reshape(total, srv.h + 2 * srv.n_kv, srv.d)
        cu = np.concatenate([[0], np.cumsum(new)])
        for r in range(n):
            hist_k[r] = np.concatenate([hist_k[r], kk[cu[r]:cu[r + 1], srv.h:srv.h + srv.n_kv]])
            hist_v[r] = np.concatenate([hist_v[r], kk[cu[r]:cu[r + 1], srv.h + srv.n_kv:]])
        kv = [len(x) for x in hist_k]
        assert srv.kv.tolist() == kv and srv.cu.tolist() == cu.tolist()
        got = srv.out.double().cpu().numpy()
        want, mine, mag, sco = po.attend(srv.q[:total].double().cpu().numpy(), hist_k, hist_v, cu, kv, srv.d ** -0.5, 1)
        tol = 2.0 ** -8 * 1.01 * (np.abs(want) + mag) + mag * (2 * srv.d * 2.0 ** -24 * sco[..., None] + 2.0 ** -18)
        assert (np.abs(got[:total] - want) <= tol + 2.0 ** -24).all()
        np.testing.assert_array_equal(got[total:], before[total:].double().cpu().numpy())
        lg = srv.logits.double().cpu().numpy()
        nxt = srv.next.cpu().numpy()
        assert nxt.tolist() == [po.sample(lg[r], 1.0, 0, float(np.float32(0.9)), 0.0, float(u[r])) for r in range(n)]
    live = [int(x) for r in range(n) for x in srv.table[r, : -(-kv[r] // 16)].tolist()]
    assert len(set(live)) == len(live) and int(srv.n_free) == srv.n_pages - len(live)
