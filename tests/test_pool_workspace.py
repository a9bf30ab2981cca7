"""The workspace of kg_pool_attend_dev, without a device: it holds what the CTAs that fit a B200 at a time write, two on
each of 148 SMs for the short requests and one for the long ones, and no more than the header says."""
import pytest

A16 = 1 << 20


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n_head,n_kv,total_q", [(1, 1, 1), (8, 8, 16), (8, 2, 16), (8, 2, 17), (64, 1, 1), (64, 1, 2), (32, 8, 1 << 20)])
def test_workspace_bytes(kg, d, n_head, n_kv, total_q):
    pool = kg.page_pool(A16, A16 + 16 * n_kv * d * 2, 8, 16, n_kv, d)
    got = kg.CudaBackend.pool_attend_bytes(pool, 4, n_head, total_q)
    rows = total_q * (n_head // n_kv)
    short = min(-(-rows // 16) * 16, 64) * (d + 2) * 4 + 16  # an item's sums, (maximum, sum) and what it is
    long = (256 * (d + 2) * 4 + 16) * (rows > 64)
    assert 2 * (296 * short + 148 * long) <= got <= 2 * (320 * short + 160 * long) <= 64e6
