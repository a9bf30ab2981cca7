"""kg_sample_logits_dev on f16 logits of the largest vocabularies, and on rows so even that the step which holds a cut has
more entries than the first CTA sorts: there the cut is found by bisection, without the key bits that a type does not use."""
import numpy as np
import pytest

from test_gpu_logits import _check

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be(kg):
    b = kg.CudaBackend(kg.micro_config())
    yield b
    b.pool_status()
    b.close()


@pytest.mark.parametrize("vocab", [131072, 262144])
def test_largest_vocabularies(be, vocab):
    rng = np.random.default_rng(vocab + 1)
    x = (rng.standard_normal((6, vocab)) * 2).astype(np.float32)
    _check(be, x, "f16", [1.0, 0.7, 1.3, 0.0, 1.0, 5.0], [0, 0, 50, 0, 20000, 0], [1.0, 0.9, 0.95, 1.0, 0.5, 0.999], [0, 0, 0, 0, 0.01, 0],
           rng.random(6))


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("width", [0.005, 0.02, 6e-5])
def test_crowded_steps(be, dt, width):
    """All logits within one or a few steps of the histogram (in f16 some below 2^-14, where it holds fewer bits)."""
    rng = np.random.default_rng(int(width * 1e6))
    x = (rng.random((8, 50000)) * width).astype(np.float32)
    x[4:] = -x[4:]
    _check(be, x, dt, None, [7, 300, 5000, 40000, 1, 4097, 20000, 0], None, None, rng.random(8))
    _check(be, x, dt, None, None, [0.1, 0.5, 0.9, 0.999, 0.01, 0.3, 0.7, 1.0], None, rng.random(8))
    _check(be, x, dt, [0.7] * 8, [0, 30000, 9000, 0, 49999, 100, 12000, 40000], [0.9, 0.5, 0.2, 1.0, 0.95, 0.8, 0.6, 0.4], [0.0, 0.99] * 4,
           rng.random(8))
