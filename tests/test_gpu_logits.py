"""kg_sample_logits_dev against the definition in python floats: whole numbers, equal on every row."""
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


def _draw(be, x, dt, temp, top_k, top_p, min_p, u, pad=0, shift=0, stream=None):
    """Tokens of rows x (numpy f32, rounded to dt here) and the values the device saw."""
    import torch
    td = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[dt]
    n, v = x.shape
    room = torch.full((n * (v + pad) + shift,), float("nan"), dtype=td, device="cuda")
    room[shift:].view(n, v + pad)[:, :v] = torch.from_numpy(x).to(td).cuda()
    lg = room[shift:].view(n, v + pad)[:, :v]
    f = lambda y, t: None if y is None else torch.as_tensor(np.asarray(y), dtype=t).cuda()  # noqa: E731
    t_, k_, p_, m_, u_ = f(temp, torch.float32), f(top_k, torch.int32), f(top_p, torch.float32), f(min_p, torch.float32), f(u, torch.float32)
    out = torch.full((n + 1,), 777, dtype=torch.int32, device="cuda")
    ptr = lambda y: None if y is None else y.data_ptr()  # noqa: E731
    be.sample_logits_dev(n, v, dt, lg.data_ptr(), v + pad, ptr(t_), ptr(k_), ptr(p_), ptr(m_), ptr(u_), out.data_ptr(), stream)
    torch.cuda.synchronize()
    assert int(out[n]) == 777
    return out[:n].cpu().numpy(), lg.double().cpu().numpy()


def _check(be, x, dt, temp, top_k, top_p, min_p, u, **kw):
    got, lg = _draw(be, x, dt, temp, top_k, top_p, min_p, u, **kw)
    n = x.shape[0]
    of = lambda y, i, d: d if y is None else float(np.float32(y[i]))  # noqa: E731
    want = [po.sample(lg[i], of(temp, i, 1.0), int(of(top_k, i, 0)), of(top_p, i, 1.0), of(min_p, i, 0.0), float(np.float32(u[i])))
            for i in range(n)]
    assert got.tolist() == want


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("vocab,pad,shift", [(1, 0, 0), (2, 1, 0), (27, 0, 1), (1000, 3, 0), (4097, 0, 3), (32000, 0, 0), (50001, 1, 1)])
def test_mixed_rows(be, dt, vocab, pad, shift):
    rng = np.random.default_rng(vocab)
    n = 24
    x = (rng.standard_normal((n, vocab)) * rng.choice([0.3, 2.0, 6.0], (n, 1))).astype(np.float32)
    temp = rng.uniform(0.3, 1.7, n)
    temp[5] = 0.0
    top_k = rng.choice([0, 1, 2, 40, 300, 5000, 10**6], n)
    top_p = rng.choice([1.0, 0.9, 0.5, 0.99, 0.05, 0.0], n)
    min_p = rng.choice([0.0, 0.0, 0.05, 0.3], n)
    u = rng.random(n)
    _check(be, x, dt, temp, top_k, top_p, min_p, u, pad=pad, shift=shift)
    _check(be, x, dt, None, None, None, None, u, pad=pad, shift=shift)
    _check(be, x, dt, None, top_k, None, None, u, pad=pad, shift=shift)
    _check(be, x, dt, temp, None, top_p, None, u, pad=pad, shift=shift)
    _check(be, x, dt, None, None, None, min_p, u, pad=pad, shift=shift)


@pytest.mark.parametrize("vocab", [131072, 262144])
def test_largest_vocabularies(be, vocab):
    rng = np.random.default_rng(vocab)
    x = (rng.standard_normal((6, vocab)) * 2).astype(np.float32)
    for dt in ("f32", "bf16"):
        _check(be, x, dt, [1.0, 0.7, 1.3, 0.0, 1.0, 5.0], [0, 0, 50, 0, 20000, 0], [1.0, 0.9, 0.95, 1.0, 0.5, 0.999], [0, 0, 0, 0, 0.01, 0],
               rng.random(6))


def test_every_value_equal(be):
    n, vocab = 12, 5003
    x = np.full((n, vocab), -3.25, np.float32)
    u = np.linspace(0, 1 - 2.0 ** -24, n)
    _check(be, x, "bf16", None, None, None, None, u)
    _check(be, x, "bf16", None, [7] * n, None, None, u)
    _check(be, x, "f32", None, [700] * n, [0.5] * n, None, u)
    _check(be, x, "f16", None, None, [0.25] * n, [1.0] * n, u)


def test_few_values_many_ties(be):
    rng = np.random.default_rng(8)
    x = rng.choice([0.0, -0.0, 1.0, 2.0, -5.0], (16, 20011)).astype(np.float32)
    _check(be, x, "f32", None, rng.choice([1, 100, 5000, 0], 16), rng.choice([0.3, 0.9, 1.0], 16), None, rng.random(16))
    _check(be, x, "bf16", np.full(16, 0.5), None, rng.choice([0.3, 0.9, 0.97], 16), None, rng.random(16))


def test_masked_infinite_and_missing_values(be):
    inf, nan, low = np.inf, np.nan, np.finfo(np.float32).min
    rows = [[-inf] * 5, [nan] * 5, [nan, -inf, 1.0, nan, -inf], [inf, 1.0, inf, -inf, nan], [low, low, -inf, low, low], [low, 0.0, nan, low, 3e38],
            [-inf, -inf, -inf, -inf, -7.0], [1.0, inf, 2.0, nan, 3.0], [1e38, -1e38, 3e38, 0.0, 2.9e38], [-0.0, 0.0, -inf, -inf, -inf]]
    x = np.array(rows, np.float32)
    for u in (0.0, 0.4, 0.999):
        n = len(rows)
        _check(be, x, "f32", None, None, None, None, [u] * n)
        _check(be, x, "f32", [0.0] * n, None, None, None, [u] * n)
        _check(be, x, "f32", [0.5] * n, [2] * n, [0.9] * n, [0.1] * n, [u] * n)
        _check(be, x, "f32", [1e30] * n, None, [0.9] * n, None, [u] * n)
        _check(be, x, "f32", [1e-30] * n, None, [0.9] * n, None, [u] * n)
        _check(be, x, "bf16", None, None, [0.5] * n, None, [u] * n)
    big = np.full((3, 40000), -np.inf, np.float32)
    big[0, 39999], big[1, [5, 39000]] = -2.0, [1.0, 0.5]
    _check(be, big, "f32", None, [50] * 3, [0.95] * 3, None, [0.7] * 3)
    _check(be, big, "bf16", None, None, None, None, [0.7] * 3)


def test_parameters_at_their_ends(be):
    rng = np.random.default_rng(2)
    x = np.tile(rng.standard_normal((1, 3000)).astype(np.float32), (10, 1))
    u = rng.random(10)
    got, lg = _draw(be, x, "f32", [-1.0, np.nan, 0.0, np.inf, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0], [0, 0, 0, 0, -5, 2**31 - 1, 0, 0, 0, 0],
                    [1, 1, 1, 1, 1, 1, -1.0, np.nan, 2.0, 1.0], [0, 0, 0, 0, 0, 0, 0, 0, np.nan, 2.0], u)
    top = int(lg[0].argmax())
    plain = [po.sample(lg[0], 1.0, 0, 1.0, 0.0, float(np.float32(y))) for y in u]
    flat = int(np.floor(float(np.float32(u[3])) * 3000))  # an infinite temperature: every token alike
    assert got.tolist() == [top, top, top, flat, plain[4], plain[5], top, plain[7], plain[8], top]
    # numbers outside [0, 1)
    got, _ = _draw(be, x[:4], "f32", None, [3] * 4, None, None, [-0.5, 1.0, 7.0, np.nan])
    first, last = min(np.argsort(-lg[0])[:3]), max(np.argsort(-lg[0])[:3])
    assert got.tolist() == [first, last, last, first]


def test_one_row_many_numbers(be):
    """The share of each token over a fine grid of numbers is its probability: the running sum is the right one."""
    n = 4000
    x = np.tile(np.log(np.array([[0.1, 0.2, 0.05, 0.4, 0.25]])).astype(np.float32), (n, 1))
    got, _ = _draw(be, x, "f32", None, None, None, None, (np.arange(n) + 0.5) / n)
    assert (np.diff(got) >= 0).all()
    np.testing.assert_allclose(np.bincount(got, minlength=5) / n, [0.1, 0.2, 0.05, 0.4, 0.25], atol=1.01 / n)


def test_graph_and_stream(be):
    import torch
    rng = np.random.default_rng(3)
    x = torch.from_numpy(rng.standard_normal((32, 32000)).astype(np.float32)).cuda()
    u, p = torch.rand(32, device="cuda"), torch.full((32,), 0.9, device="cuda")
    out = torch.zeros(32, dtype=torch.int32, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    call = lambda: be.sample_logits_dev(32, 32000, "f32", x.data_ptr(), 32000, None, None, p.data_ptr(), None, u.data_ptr(),  # noqa: E731
                                        out.data_ptr(), s.cuda_stream)
    with torch.cuda.stream(s):
        call()
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            call()
        u.copy_(torch.rand(32, device="cuda"))
        out.zero_()
        g.replay()
    s.synchronize()
    lg, uu = x.double().cpu().numpy(), u.cpu().numpy()
    assert out.tolist() == [po.sample(lg[i], 1.0, 0, float(np.float32(0.9)), 0.0, float(uu[i])) for i in range(32)]
