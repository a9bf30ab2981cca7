"""The attention over a page pool when its device-side waits run out: the kernels end, kg_pool_status says so, and the
calls that follow are right. The limit is a few clock cycles, so that waits for loads, scores, probabilities and values
run out in the middle of a part."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


class Call:
    def __init__(self, kg, be, reqs, n_head, n_kv, d, dt, causal):
        import torch
        td = {"bf16": torch.bfloat16, "f16": torch.float16}[dt]
        g = torch.Generator(device="cuda").manual_seed(len(reqs))
        page, n = 16, len(reqs)
        need = [-(-kv // page) for _, kv in reqs]
        self.m = torch.randn(sum(need), 2, page, n_kv, d, generator=g, device="cuda").to(td)
        self.pool = kg.page_pool(self.m.data_ptr(), self.m[0, 1].data_ptr(), sum(need), page, n_kv, d, dt)
        width, at = max(need), 0
        table = np.full((n, width), -1)
        for r in range(n):
            table[r, :need[r]] = np.arange(at, at + need[r])
            at += need[r]
        i32 = lambda x: torch.as_tensor(np.asarray(x), dtype=torch.int32).cuda()  # noqa: E731
        self.table, self.kv = i32(table), i32([kv for _, kv in reqs])
        self.cu = i32(np.concatenate([[0], np.cumsum([q for q, _ in reqs])]))
        total = int(self.cu[-1])
        self.q = torch.randn(total + 3, n_head, d, generator=g, device="cuda").to(td)
        self.out = torch.full_like(self.q, 7.0)
        self.ws = torch.zeros(be.pool_attend_bytes(self.pool, n, n_head, total), dtype=torch.uint8, device="cuda")
        self.args = (n, n_head, total)
        self.d, self.causal, self.be, self.width, self.total = d, causal, be, width, total

    def __call__(self):
        q, o = self.q, self.out
        self.be.pool_attend_dev(self.pool, *self.args, self.cu.data_ptr(), self.kv.data_ptr(), self.table.data_ptr(), self.width, q.data_ptr(),
                                q.stride(0), q.stride(1), o.data_ptr(), o.stride(0), o.stride(1), self.d ** -0.5, self.causal,
                                self.ws.data_ptr(), self.ws.numel())


CASES = [
    ([(1, 3000), (1, 40), (4, 900)], 8, 2, 128, "bf16", 1),   # short requests
    ([(1, 700)] * 60, 12, 12, 64, "f16", 1),
    ([(300, 2000)], 8, 2, 128, "bf16", 1),                     # long ones
    ([(90, 90), (200, 1500), (65, 70)], 4, 4, 64, "f16", 0),
    ([(400, 900), (1, 2500), (1, 10), (70, 3000)], 8, 1, 128, "f16", 1),  # both
]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_waits_that_run_out_end_the_call(kg, case):
    import torch
    be = kg.CudaBackend(kg.micro_config())
    lib = kg.lib()
    assert lib.kg_selftest_pool_wait(be._h, -1) == -1 and lib.kg_selftest_pool_wait(be._h, (1 << 30) + 1) == -1
    call = Call(kg, be, *CASES[case])
    call()
    be.pool_status()
    want = call.out.clone()
    ran_out = 0
    for limit in (1, 200, 1000, 2000, 4000, 8000, 16000, 40000):
        assert lib.kg_selftest_pool_wait(be._h, limit) == 0
        for _ in range(3):
            call()
        try:
            be.pool_status()
        except kg.KgError as e:
            assert e.status == -4 and "exceeded" in str(e)  # KG_ERR_TIMEOUT
            ran_out += 1
        assert (call.out[call.total:] == 7).all()
        assert lib.kg_selftest_pool_wait(be._h, 0) == 0
        call()
        be.pool_status()
        assert torch.equal(call.out, want)
    assert ran_out > 0
    be.close()


def test_a_rejected_argument_does_not_hide_a_wait_that_ran_out(kg):
    import torch
    be = kg.CudaBackend(kg.micro_config())
    lib = kg.lib()
    call = Call(kg, be, *CASES[4])
    rows = torch.zeros(1, 1, call.d, device="cuda")
    slot = torch.full((1,), 1 << 20, dtype=torch.int32, device="cuda")  # past the pool
    cu = call.cu.clone()

    def reject_store():
        be.pool_store_dev(call.pool, 1, slot.data_ptr(), "f32", rows.data_ptr(), rows.data_ptr(), call.d, call.d)

    def reject_lengths():
        call.cu.copy_(cu + call.total)
        call()
        call.cu.copy_(cu)

    def reject_table(reqs):
        keep = call.table.clone()
        call.table[reqs, 0] = -5
        call()
        call.table.copy_(keep)

    for reject in (reject_store, reject_lengths, lambda: reject_table(1), lambda: reject_table(0)):
        lib.kg_selftest_pool_wait(be._h, 1)
        call()
        lib.kg_selftest_pool_wait(be._h, 0)
        reject()
        with pytest.raises(kg.KgError, match="exceeded") as e:
            be.pool_status()
        assert e.value.status == -4
        reject()
        with pytest.raises(kg.KgError, match="rejected"):
            be.pool_status()
        be.pool_status()
    be.close()
