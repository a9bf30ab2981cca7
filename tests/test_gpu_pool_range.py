"""Attention over the page pool where the numbers' range counts: probabilities far below a row's largest, which f16 holds
only near its own upper end, and scores so large that f32 has no number near them. Against 64 bits, in both kernels
(requests of at most 64 rows a K/V head, and longer ones)."""
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


def _shared(kg, be, k, v, q, n_req, dt, scale, causal, page=64):
    """`n_req` requests of q's rows each over the same pages: (rows of all requests, their 64-bit values, tolerances).
    k, v: [positions][kv heads][d], q: [rows][heads][d], numpy."""
    import torch
    td = {"bf16": torch.bfloat16, "f16": torch.float16}[dt]
    kv, n_kv, d = k.shape
    rows, heads, _ = q.shape
    pages = -(-kv // page)
    m = torch.full((pages, 2, page, n_kv, d), float("nan"), dtype=td, device="cuda")
    for i, x in enumerate((k, v)):
        y = torch.full((pages * page, n_kv, d), float("nan"), dtype=td)
        y[:kv] = torch.from_numpy(x).to(td)
        m[:, i] = y.view(pages, page, n_kv, d).cuda()
    k, v, q = (torch.from_numpy(x).to(td) for x in (k, v, q))
    pool = kg.page_pool(m.data_ptr(), m[0, 1].data_ptr(), pages, page, n_kv, d, dt)
    qd = q.cuda().repeat(n_req, 1, 1)
    out = torch.full_like(qd, 7.0)
    i32 = dict(dtype=torch.int32, device="cuda")
    cu, kvd = torch.arange(n_req + 1, **i32) * rows, torch.full((n_req,), kv, **i32)
    table = torch.arange(pages, **i32).repeat(n_req, 1)
    ws = torch.full((be.pool_attend_bytes(pool, n_req, heads, n_req * rows),), 0xFF, dtype=torch.uint8, device="cuda")
    be.pool_attend_dev(pool, n_req, heads, n_req * rows, cu.data_ptr(), kvd.data_ptr(), table.data_ptr(), pages, qd.data_ptr(), qd.stride(0),
                       qd.stride(1), out.data_ptr(), out.stride(0), out.stride(1), scale, causal, ws.data_ptr(), ws.numel())
    torch.cuda.synchronize()
    be.pool_status()
    want, _, mag, sco = po.attend(q.double().numpy(), [k.double().numpy()], [v.double().numpy()], [0, rows], [kv], scale, causal)
    # one rounding of the result and one of every probability, half a step each, f32 scores (d products) and 2^-18 for exp
    # and the running sums, as for ordinary batches
    half = torch.finfo(td).eps / 2
    tol = half * np.abs(want) * 1.01 + mag * (half * 1.01 + 2 * d * 2.0 ** -24 * sco[..., None] + 2.0 ** -18) + 2.0 ** -24
    return out.double().cpu().numpy().reshape(n_req, rows, heads, d), want, tol


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("rows,n_req,positions,nats,d", [
    (1, 1, 65536, 17.3, 64), (5, 1, 16384, 16.2, 128), (1, 300, 2000, 15.0, 128), (4, 9, 3001, 17.0, 64),  # short
    (40, 1, 65536, 17.3, 64), (150, 1, 16384, 16.2, 128), (40, 80, 2000, 15.0, 128), (70, 9, 3001, 17.0, 64),  # long
])
@pytest.mark.parametrize("at", ["first", "middle", "last"])
def test_a_far_peak_and_a_flat_rest(kg, be, dt, rows, n_req, positions, nats, d, at):
    """One position takes nearly the whole weight and has no value (an attention sink); the result is the flat rest's share,
    whose probabilities lie 2^-21 to 2^-25 below the largest."""
    rng = np.random.default_rng(rows + positions)
    k, v = np.zeros((positions, 1, d)), rng.uniform(0.5, 1.5, (positions, 1, d))
    peak = {"first": 0, "middle": positions // 2, "last": positions - rows}[at]  # every row attends it
    k[peak, 0, 0], v[peak] = nats * d ** 0.5 / 8, 0.0
    q = rng.standard_normal((rows, 2, d))
    q[..., 0] = 8.0
    got, want, tol = _shared(kg, be, k, v, q, n_req, dt, d ** -0.5, 1)
    assert (np.abs(got - want) <= tol).all(), (np.abs(got - want) / tol).max()


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 70])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_scores_past_the_whole_numbers_of_f32(kg, be, dt, rows, sign):
    """Equal scores of 2^18 to 2^29: every weight is the same, whatever is subtracted from the scores must not make one
    of them overflow."""
    d, positions = 64, 300
    rng = np.random.default_rng(5)
    v = rng.uniform(0.5, 1.5, (positions, 1, d))
    q = np.zeros((rows, 1, d))
    q[..., 0] = 2.0 ** 14
    for e in range(4, 16):
        for f in (1.0, 1.375):
            k = np.zeros((positions, 1, d))
            k[..., 0] = sign * f * 2.0 ** e
            got, want, tol = _shared(kg, be, k, v, q, 1, dt, 1.0, 0)
            assert (np.abs(got - want) <= tol).all(), (e, f)


@pytest.mark.parametrize("fits", [True, False])
def test_a_plan_with_room_for_two_billion_tokens(be, fits):
    """The largest max_tokens (26 GB of token entries): the padding ends where the entries do."""
    import torch
    m = 2**31 - 1
    i32 = dict(dtype=torch.int32, device="cuda")
    slots, req, pos = (torch.full((m + 9,), 777, **i32) for _ in range(3))
    cached, new, table = torch.tensor([5, 0], **i32), torch.tensor([3, 20 if fits else -1], **i32), torch.zeros(2, 4, **i32)
    free, n_free, left = torch.arange(1, 8, **i32), torch.tensor([7], **i32), torch.zeros(1, **i32)
    cu, kv, status = torch.zeros(3, **i32), torch.zeros(2, **i32), torch.zeros(1, **i32)
    p = lambda x: x.data_ptr()  # noqa: E731
    be.pool_plan_dev(16, 8, 2, p(cached), p(new), p(table), 4, p(free), p(n_free), p(left), m, p(cu), p(kv), p(slots), p(req), p(pos), p(status))
    torch.cuda.synchronize()
    total = 23 if fits else 0
    assert int(status) == (0 if fits else -1) and cu.tolist() == ([0, 3, 23] if fits else [0, 0, 0])
    for x in (slots, req, pos):
        assert (x[:total] >= 0).all() and (x[m:] == 777).all()
        for at in range(total, m, 1 << 28):
            assert (x[at:min(at + (1 << 28), m)] == -1).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("reqs,n_head,n_kv,d", [
    ([(2, 9000), (3, 2), (1, 40)], 4, 2, 128),   # short: positions split over the device, whole, rows before position 0
    ([(1, 900)] * 400, 2, 2, 64),
    ([(100, 9000), (70, 30), (80, 80)], 4, 2, 128),  # long
    ([(90, 300)] * 60, 2, 1, 64),
])
def test_a_query_that_is_not_a_number(kg, be, bad, reqs, n_head, n_kv, d):
    """Its rows come out as NaN wherever the items are cut, a row that attends nothing as zeros, the others as they are."""
    import torch
    page, pages = 16, 600
    g = torch.Generator(device="cuda").manual_seed(3)
    m = torch.randn(pages, 2, page, n_kv, d, generator=g, device="cuda").half()
    pool = kg.page_pool(m.data_ptr(), m[0, 1].data_ptr(), pages, page, n_kv, d, "f16")
    i32 = dict(dtype=torch.int32, device="cuda")
    q_len, kv = [r[0] for r in reqs], [r[1] for r in reqs]
    cu, kvd = torch.tensor([0] + list(np.cumsum(q_len)), **i32), torch.tensor(kv, **i32)
    table = torch.arange(pages, **i32).repeat(len(reqs), 1)
    total = sum(q_len)
    q = torch.randn(total, n_head, d, generator=g, device="cuda").half()
    ws = torch.full((be.pool_attend_bytes(pool, len(reqs), n_head, total),), 0xFF, dtype=torch.uint8, device="cuda")

    def run(q):
        out = torch.full_like(q, 7.0)
        be.pool_attend_dev(pool, len(reqs), n_head, total, cu.data_ptr(), kvd.data_ptr(), table.data_ptr(), pages, q.data_ptr(), q.stride(0),
                           q.stride(1), out.data_ptr(), out.stride(0), out.stride(1), d ** -0.5, 1, ws.data_ptr(), ws.numel())
        torch.cuda.synchronize()
        be.pool_status()
        return out
    good = run(q)
    hit = torch.zeros(total, n_head, dtype=torch.bool, device="cuda")
    hit[::3, n_head - 1] = True
    hit[1::5, 0] = True
    hit[cu[:-1].long()] = True
    none = torch.cat([torch.arange(a, device="cuda") - a + b < 0 for a, b in reqs])[:, None].expand_as(hit)  # attends nothing
    q2 = q.clone()
    q2[..., 3] = torch.where(hit, torch.full_like(q2[..., 3], bad), q2[..., 3])
    got = run(q2)
    assert (got[hit & ~none].isnan()).all()
    assert (got[none] == 0).all() and torch.equal(got[~hit], good[~hit])


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("rows", [2, 70])
def test_large_scores_of_any_bits(kg, be, dt, rows):
    """Scores whose product with the scale has more bits than f32: one position of each row is far above the others, so that
    the row is that position's value. Requests of more than 64 rows promise it up to 2^26."""
    import torch
    d, positions = 64, 200
    rng = np.random.default_rng(11)
    half = torch.finfo({"bf16": torch.bfloat16, "f16": torch.float16}[dt]).eps / 2
    for e in range(9):
        for scale in (0.001, 0.3, 1.0, 7.3, 30.0):
            if rows > 64 and 2.0 ** (7 + e + 15) * scale > 2.0 ** 26:
                continue
            k = np.zeros((positions, 1, d))
            k[:, 0, 0] = rng.uniform(0.1, 0.5, positions) * 2.0 ** (6 + e)
            k[rng.integers(0, positions), 0, 0] = rng.uniform(1.0, 2.0) * 2.0 ** (6 + e)
            q = np.zeros((rows, 2, d))
            q[..., 0] = rng.uniform(0.5, 1.0, (rows, 2)) * 2.0 ** 15
            v = rng.uniform(0.5, 1.5, (positions, 1, d))
            got, want, _ = _shared(kg, be, k, v, q, 1, dt, scale, 0)
            # the one probability is rounded and divided by itself unrounded, then the result: half a step each
            assert (np.abs(got - want) <= 2 * half * 1.01 * np.abs(want)).all(), (e, scale, np.abs(got - want).max())


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("rows,positions,d", [(1, 5000, 64), (3, 700, 128), (70, 5000, 128), (200, 1500, 64)])
@pytest.mark.parametrize("span", [3.0, 30.0, -30.0, 300.0])
def test_rising_and_falling_scores(kg, be, dt, rows, positions, d, span):
    """The running maximum grows all the way, by little or by much in a unit, or is the first position's; rows differ in how
    steeply."""
    rng = np.random.default_rng(rows)
    k, q = rng.standard_normal((positions, 2, d)) * 0.2, rng.standard_normal((rows, 4, d)) * 0.2
    k[..., 0] = np.linspace(-0.5, 0.5, positions)[:, None] * span
    q[..., 0] = d ** 0.5 * rng.uniform(0.1, 1.0, (rows, 4))
    v = rng.standard_normal((positions, 2, d)) + 1.0
    got, want, tol = _shared(kg, be, k, v, q, 2, dt, d ** -0.5, 1)
    assert (np.abs(got - want) <= tol).all(), (np.abs(got - want) / tol).max()
    again, _, _ = _shared(kg, be, k, v, q, 2, dt, d ** -0.5, 1)
    np.testing.assert_array_equal(got, again)
