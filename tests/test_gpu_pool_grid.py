"""Attention over the page pool: every type, head size and page size in the long requests' kernel (more than 64 rows a K/V
head), and the long batches of test_gpu_pool.py in f16."""
import itertools

import pytest

from test_gpu_pool import _attend_case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be(kg):
    b = kg.CudaBackend(kg.micro_config())
    yield b
    b.pool_status()
    b.close()


@pytest.mark.parametrize("d,page,dt,causal", list(itertools.product([64, 128], [16, 32, 64, 128], ["bf16", "f16"], [1, 0])))
def test_long_and_short_requests(kg, be, d, page, dt, causal):
    _attend_case(kg, be, [(70, 300), (33, 40), (1, 129), (0, 5), (150, 150), (40, 8), (3, 1000), (65, 1029)], 4, 2, d, page, dt, causal, pad=2,
                 seed=d + page)


@pytest.mark.parametrize("reqs,n_head,n_kv,d,page", [
    ([(130, 3000)], 8, 2, 128, 16),
    ([(300, 300), (1, 900), (257, 700)], 4, 4, 128, 16),
    ([(600, 600), (128, 128), (129, 1290)], 2, 1, 64, 64),
    ([(90, 1000), (43, 1000), (1, 77)], 6, 2, 128, 128),
    ([(70, 333), (52, 52)], 10, 2, 64, 16),
    ([(20, 9000)], 8, 1, 128, 16),
    ([(2, 50), (3, 700), (9, 130)], 64, 1, 128, 16),
    ([(129, 20), (300, 150), (80, 0)], 2, 1, 128, 16),
])
@pytest.mark.parametrize("spread", [1.0, 4.0])
def test_long_requests_in_f16(kg, be, reqs, n_head, n_kv, d, page, spread):
    for causal in (1, 0):
        _attend_case(kg, be, reqs, n_head, n_kv, d, page, "f16", causal, seed=len(reqs), spread=spread)
