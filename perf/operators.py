"""The serving-step operators over a caller-owned page pool, measured one by one: the plan (block tables and slot
maps from request lengths), the store of new K/V rows into pages, the attention of new tokens over the pages, and
sampling from logits. `run` computes each in elementary torch operations, or, where `own` is true, through the
framework's calls."""
import math
import os
import random
import sys

import torch

own = False

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_backend = None


def _be():
    """The library handle that a serving program keeps."""
    global _backend
    if _backend is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "katgpt-rs_b200"))
        import kgcuda
        _backend = (kgcuda, kgcuda.CudaBackend(kgcuda.micro_config()))
    return _backend


def _stream():
    return torch.cuda.current_stream().cuda_stream


# ---------------------------------------------------------------- cases

def listed():
    return [
        # one decode step of 64 sequences past a 1024-token prompt: the smallest call, bound by its latency
        dict(name="plan decode", op="plan", n_req=64, new_lo=1, new_hi=1, old_lo=1024, old_hi=1200, page=16, mix=1, pad=0),
        # a prefill batch of ragged prompts, some continuing a cached prefix
        dict(name="plan prefill", op="plan", n_req=512, new_lo=0, new_hi=255, old_lo=0, old_hi=4000, page=16, mix=2, pad=37),
        # one new row of each of 256 sequences, 32 heads of 128
        dict(name="store decode", op="store", rows=256, n_kv=32, d=128, page=16, src="bf16", dt="bf16", pages=2048, skip=0.0),
        # f32 rows of a fused QKV product of 12 heads of 64: 16 prompts of 1024 tokens, with padding rows
        dict(name="store prefill", op="store", rows=16500, n_kv=12, d=64, page=16, src="f32", dt="bf16", pages=2048, skip=0.01),
        # decode of 64 sequences past a 1024-token prompt, 12 heads of 64, every head with its own K/V
        dict(name="decode 12x64", op="attend", n_req=64, q_lo=1, q_hi=1, kv_lo=1025, kv_hi=1200, n_head=12, n_kv=12, d=64,
             page=16, dt="bf16", causal=1, mix=3, pad=0),
        # decode over long contexts of unlike length, 8 K/V heads for 32 query heads
        dict(name="decode long grouped", op="attend", n_req=32, q_lo=1, q_hi=1, kv_lo=300, kv_hi=16384, n_head=32, n_kv=8, d=128,
             page=16, dt="bf16", causal=1, mix=4, pad=0),
        # decode of 64 sequences near 4096 positions, 32 heads of 128: the widest cache rows
        dict(name="decode 32x128", op="attend", n_req=64, q_lo=1, q_hi=1, kv_lo=4096, kv_hi=4223, n_head=32, n_kv=32, d=128,
             page=16, dt="bf16", causal=1, mix=5, pad=0),
        # draft paths being verified: five new tokens of each of 16 sequences, f16
        dict(name="verify drafts", op="attend", n_req=16, q_lo=5, q_hi=5, kv_lo=1500, kv_hi=4200, n_head=32, n_kv=8, d=128,
             page=16, dt="f16", causal=1, mix=6, pad=0),
        # one chunk of a long prompt over what earlier chunks left in the cache
        dict(name="chunk of a prompt", op="attend", n_req=1, q_lo=2048, q_hi=2048, kv_lo=18000, kv_hi=18000, n_head=32, n_kv=8,
             d=128, page=16, dt="bf16", causal=1, mix=7, pad=0),
        # ragged prompts of 16 heads of 128 from position 0, with single tokens among them
        dict(name="ragged prompts", op="attend", n_req=9, q_lo=1, q_hi=4096, kv_lo=0, kv_hi=300, n_head=16, n_kv=16, d=128,
             page=16, dt="bf16", causal=1, mix=8, pad=5),
        # every request with its own sampling parameters, f32 logits over 32000 words
        dict(name="sample mixed", op="sample", rows=64, vocab=32000, dt="f32", kind="mixed", spread=2.5, pad=0),
        # nucleus sampling of a large batch over a vocabulary of 131072, bf16 logits (many ties)
        dict(name="sample nucleus", op="sample", rows=256, vocab=131072, dt="bf16", kind="nucleus", spread=2.0, pad=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "store", "attend", "attend", "attend", "sample"])
    page = rng.choice([16, 16, 32, 64, 128])
    mix = rng.randrange(1 << 20)
    if op == "plan":
        n_req = _log(rng, 1, 1024)
        new_hi = _log(rng, 1, max(1, 60000 // n_req))
        return dict(op=op, n_req=n_req, new_lo=rng.choice([0, 1, new_hi]), new_hi=new_hi, old_lo=0, old_hi=_log(rng, 1, 4000),
                    page=page, mix=mix, pad=rng.choice([0, 1, 300]))
    if op == "store":
        n_kv, d = rng.choice([1, 2, 3, 8, 12, 16]), rng.choice([64, 128])
        return dict(op=op, rows=_log(rng, 1, 16000 * 768 // (n_kv * d)), n_kv=n_kv, d=d, page=page,
                    src=rng.choice(["f32", "bf16", "f16"]), dt=rng.choice(["bf16", "f16"]), pages=400000 // (n_kv * page),
                    skip=rng.choice([0.0, 0.02]))
    if op == "sample":
        vocab = _log(rng, 100, 131072)
        return dict(op=op, rows=min(_log(rng, 1, 256), 256), vocab=vocab, dt=rng.choice(["f32", "bf16", "f16"]),
                    kind=rng.choice(["mixed", "nucleus", "plain", "topk"]), spread=rng.choice([0.5, 2.0, 4.0]), pad=rng.choice([0, 8]))
    n_kv, d = rng.choice([1, 2, 4, 8]), rng.choice([64, 128])
    group = rng.choice([1, 2, 3, 4, 5, 6, 8, 16])
    n_req = _log(rng, 1, 48)
    form = rng.choice(["decode", "few", "chunk"])
    q_hi = 1 if form == "decode" else rng.randint(2, 17) if form == "few" else _log(rng, 20, max(21, 4000 // n_req))
    kv_lo, kv_hi = 0, _log(rng, 1, 16384 if n_req < 8 else 65536 // n_req)
    heads = n_kv * group
    while n_req * heads * q_hi * (q_hi + kv_hi) > 1.0e9:  # no dearer than the listed chunk
        q_hi = max(1, q_hi // 2)
        kv_hi = max(1, kv_hi // 2)
    return dict(op=op, n_req=n_req, q_lo=1 if form == "decode" else 0, q_hi=q_hi, kv_lo=kv_lo, kv_hi=kv_hi, n_head=heads, n_kv=n_kv,
                d=d, page=page, dt=rng.choice(["bf16", "bf16", "f16"]), causal=rng.choice([1, 1, 1, 0]), mix=mix,
                pad=rng.choice([0, 3]))


def _lengths(case):
    """New and cached lengths of every request: the case's own, whatever the seed of its values."""
    rng = random.Random(case["mix"])
    n = case["n_req"]
    if case["op"] == "plan":
        return [(rng.randint(case["new_lo"], case["new_hi"]), rng.randint(case["old_lo"], case["old_hi"])) for _ in range(n)]
    got = []
    for i in range(n):
        q = rng.randint(case["q_lo"], case["q_hi"])
        if case["q_hi"] > 64 and i % 3 == 2:  # single tokens among the chunks
            q = min(q, 1)
        kv = rng.randint(case["kv_lo"], case["kv_hi"])
        got.append((q, max(kv - q, 0) if case["kv_lo"] > 0 else kv))
    return got


def work(case):
    op = case["op"]
    if op == "plan":
        ls = _lengths(case)
        p = case["page"]
        fresh = sum(-(-(a + b) // p) - -(-b // p) for a, b in ls)
        return {"bytes": 16 * len(ls) + 8 * fresh + 12 * (sum(a for a, _ in ls) + case["pad"]), "flops": 0}
    if op == "store":
        src = 4 if case["src"] == "f32" else 2
        return {"bytes": case["rows"] * (1 - case["skip"]) * 2 * case["n_kv"] * case["d"] * (src + 2) + 4 * case["rows"], "flops": 0}
    if op == "sample":
        return {"bytes": case["rows"] * case["vocab"] * (4 if case["dt"] == "f32" else 2) + 24 * case["rows"],
                "flops": 2 * case["rows"] * case["vocab"]}
    ls = [x for x in _lengths(case) if x[0] > 0]
    pairs = sum(q * b + (q * (q + 1) // 2 if case["causal"] else q * q) for q, b in ls)
    return {"bytes": sum(2 * 2 * (q + b) * case["n_kv"] * case["d"] + 2 * 2 * q * case["n_head"] * case["d"] for q, b in ls) or 4,
            "flops": 4 * pairs * case["n_head"] * case["d"]}


# ---------------------------------------------------------------- inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dev = dict(device="cuda")
    i32 = dict(device="cuda", dtype=torch.int32)
    op = case["op"]
    s = dict(case=case)
    if op == "plan":
        ls = _lengths(case)
        p, n = case["page"], case["n_req"]
        has = [-(-b // p) for _, b in ls]
        need = [-(-(a + b) // p) for a, b in ls]
        pages = sum(need) + 100
        perm = torch.randperm(pages, generator=g, **dev).to(torch.int32)
        width = max(max(need), 1) + 3
        table = torch.full((n, width), -1, **i32)
        own_page = torch.arange(width, device="cuda")[None, :] < torch.tensor(has, device="cuda")[:, None]
        table[own_page] = perm[: sum(has)]
        total = sum(a for a, _ in ls) + case["pad"]
        s.update(new=torch.tensor([a for a, _ in ls], **i32), old=torch.tensor([b for _, b in ls], **i32), table=table, n_pages=pages,
                 free=perm[sum(has):].clone(), n_free=torch.tensor([pages - sum(has)], **i32), max_tokens=total,
                 left=torch.zeros(1, **i32), cu=torch.zeros(n + 1, **i32), kv=torch.zeros(n, **i32), slot=torch.zeros(total, **i32),
                 req=torch.zeros(total, **i32), pos=torch.zeros(total, **i32), status=torch.zeros(1, **i32))
    elif op == "store":
        rows, kvd = case["rows"], case["n_kv"] * case["d"]
        places = case["pages"] * case["page"]
        rows = min(rows, places)
        qkv = torch.randn(rows, 3 * kvd, generator=g, **dev).to(DT[case["src"]])  # [q | k | v] of a fused projection
        slots = torch.randperm(places, generator=g, **dev)[:rows].to(torch.int32)
        slots = slots.sort().values if rows > 1024 else slots  # a prompt's rows come in order
        slots[torch.rand(rows, generator=g, **dev) < case["skip"]] = -1
        s.update(k=qkv[:, kvd:2 * kvd].view(rows, case["n_kv"], case["d"]), v=qkv[:, 2 * kvd:].view(rows, case["n_kv"], case["d"]), slots=slots,
                 pool=torch.zeros(case["pages"], 2, case["page"], case["n_kv"], case["d"], dtype=DT[case["dt"]], **dev))
    elif op == "attend":
        ls = _lengths(case)
        p, n, d = case["page"], case["n_req"], case["d"]
        kv = [a + b for a, b in ls]
        need = [-(-x // p) for x in kv]
        pages = max(sum(need), 1) + 7
        width = max(max(need), 1) + 2
        perm = torch.randperm(pages, generator=g, **dev).to(torch.int32)
        table = torch.full((n, width), -1, **i32)
        table[torch.arange(width, device="cuda")[None, :] < torch.tensor(need, device="cuda")[:, None]] = perm[: sum(need)]
        total = sum(a for a, _ in ls) + case["pad"]
        pool = torch.empty(pages, 2, p, case["n_kv"], d, dtype=DT[case["dt"]], **dev)
        for i in range(0, pages, 4096):  # (in parts: the generator makes f32)
            pool[i:i + 4096] = torch.randn(pool[i:i + 4096].shape, generator=g, **dev)
        cu = [0]
        for a, _ in ls:
            cu.append(cu[-1] + a)
        q = torch.randn(max(total, 1), case["n_head"], d, generator=g, **dev).mul_(1.5).to(DT[case["dt"]])
        s.update(q=q, out=torch.zeros_like(q), pool=pool, table=table, cu=torch.tensor(cu, **i32), kv=torch.tensor(kv, **i32),
                 scale=d ** -0.5, max_q=max(max(a for a, _ in ls), 1), max_kv=max(max(need), 1) * p, space=None)
    else:
        rows, v, kind = case["rows"], case["vocab"], case["kind"]
        lg = torch.randn(rows, v + case["pad"], generator=g, **dev).mul_(case["spread"])
        r = lambda: torch.rand(rows, generator=g, **dev)  # noqa: E731
        pick = torch.arange(rows, device="cuda")
        temp, top_k, top_p, min_p = 0.5 + r(), torch.zeros(rows, **i32), torch.ones(rows, **dev), torch.zeros(rows, **dev)
        if kind in ("mixed", "topk"):
            top_k = (2 ** (r() * 10)).to(torch.int32) * ((pick % 2 == 0) | (kind == "topk"))
        if kind in ("mixed", "nucleus"):
            top_p = torch.where((pick % 3 != 0) | (kind == "nucleus"), 0.8 + 0.19 * r(), top_p)
        if kind == "mixed":
            min_p = torch.where(pick % 5 == 0, 0.02 + 0.1 * r(), min_p)
            temp = torch.where(pick % 8 == 7, 0.0, temp)
        s.update(logits=lg.to(DT[case["dt"]])[:, :v], temp=temp, top_k=top_k.to(torch.int32), top_p=top_p, min_p=min_p, u=r(),
                 out=torch.zeros(rows, **i32))
    return s


# ---------------------------------------------------------------- one pass

def run(s):
    return _RUN[s["case"]["op"]](s)


def _desc(s):
    """The pool's description, kept with the pool: [page][K rows | V rows]."""
    if "desc" not in s:
        kg, _ = _be()
        pool = s["pool"]
        s["desc"] = kg.page_pool(pool[:, 0].data_ptr(), pool[:, 1].data_ptr(), pool.shape[0], pool.shape[2], pool.shape[3], pool.shape[4],
                               s["case"]["dt"], page_stride=pool.stride(0), row_stride=pool.stride(2), head_stride=pool.stride(3))
    return s["desc"]


def _plan(s):
    p, n = s["case"]["page"], s["case"]["n_req"]
    if own:
        _, be = _be()
        be.pool_plan_dev(p, s["n_pages"], n, s["old"].data_ptr(), s["new"].data_ptr(), s["table"].data_ptr(), s["table"].shape[1],
                         s["free"].data_ptr(), s["n_free"].data_ptr(), s["left"].data_ptr(), s["max_tokens"], s["cu"].data_ptr(),
                         s["kv"].data_ptr(), s["slot"].data_ptr(), s["req"].data_ptr(), s["pos"].data_ptr(), s["status"].data_ptr(), _stream())
        return [s[k] for k in ("table", "left", "cu", "kv", "slot", "req", "pos", "status")]
    old, new, table = s["old"].long(), s["new"].long(), s["table"]
    kv = old + new
    has, need = (old + p - 1) // p, (kv + p - 1) // p
    start = torch.cumsum(need - has, 0) - (need - has)
    col = torch.arange(table.shape[1], device=table.device)[None, :]
    at = s["n_free"].long() - 1 - (start[:, None] + col - has[:, None])
    fresh = (col >= has[:, None]) & (col < need[:, None])
    table = torch.where(fresh, s["free"][at.clamp(0, s["free"].shape[0] - 1)], table)
    cu = torch.cat([new.new_zeros(1), torch.cumsum(new, 0)])
    t = torch.arange(s["max_tokens"], device=table.device)
    r = torch.searchsorted(cu[1:].contiguous(), t, right=True).clamp(max=n - 1)
    live = t < cu[-1]
    pos = old[r] + t - cu[r]
    slot = table[r, (pos // p).clamp(0, table.shape[1] - 1)].long() * p + pos % p
    i = lambda x: x.to(torch.int32)  # noqa: E731
    pad = lambda x: i(torch.where(live, x, -1))  # noqa: E731
    return [table, i(s["n_free"] - (need - has).sum()), i(cu), i(kv), pad(slot), pad(r), pad(pos), torch.zeros_like(s["status"])]


def _store(s):
    c = s["case"]
    pool, k, v, p = s["pool"], s["k"], s["v"], c["page"]
    if own:
        _, be = _be()
        be.pool_store_dev(_desc(s), k.shape[0], s["slots"].data_ptr(), c["src"], k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), _stream())
        return pool
    live = s["slots"] >= 0  # padding rows write nothing
    at = s["slots"][live].long()
    pool[at // p, 0, at % p] = k[live].float().to(pool.dtype)
    pool[at // p, 1, at % p] = v[live].float().to(pool.dtype)
    return pool


def _attend(s):
    c = s["case"]
    q, pool, p, d = s["q"], s["pool"], c["page"], c["d"]
    n, h, n_kv = c["n_req"], c["n_head"], c["n_kv"]
    if own:
        _, be = _be()
        desc = _desc(s)
        if s["space"] is None:  # the workspace that a serving program keeps
            s["space"] = torch.empty(be.pool_attend_bytes(desc, n, h, q.shape[0]), dtype=torch.uint8, device=q.device)
        be.pool_attend_dev(desc, n, h, q.shape[0], s["cu"].data_ptr(), s["kv"].data_ptr(), s["table"].data_ptr(), s["table"].shape[1],
                           q.data_ptr(), q.stride(0), q.stride(1), s["out"].data_ptr(), s["out"].stride(0), s["out"].stride(1),
                           s["scale"], c["causal"], s["space"].data_ptr(), s["space"].numel(), _stream())
        return s["out"]
    m, length = s["max_q"], s["max_kv"]
    cu, kv = s["cu"].long(), s["kv"].long()
    kvs = pool[s["table"][:, : length // p].long().clamp(min=0)]  # [n, pages, 2, p, n_kv, d]
    k = kvs[:, :, 0].reshape(n, length, n_kv, d).permute(0, 2, 3, 1).float()
    v = kvs[:, :, 1].reshape(n, length, n_kv, d).permute(0, 2, 1, 3).float()
    i = torch.arange(m, device=q.device)
    q_len = cu[1:] - cu[:-1]
    at = torch.where(i[None, :] < q_len[:, None], cu[:-1, None] + i[None, :], q.shape[0])  # the row behind the last: dropped
    qp = torch.cat([q, torch.zeros_like(q[:1])])[at].view(n, m, n_kv, h // n_kv, d).permute(0, 2, 3, 1, 4).reshape(n, n_kv, -1, d).float()
    sc = torch.matmul(qp, k).mul_(s["scale"]).view(n, n_kv, h // n_kv, m, length)
    j = torch.arange(length, device=q.device)
    last = (kv - q_len)[:, None] + i[None, :] if c["causal"] else kv[:, None].expand(n, m) - 1
    last = torch.minimum(last, kv[:, None] - 1)
    sc.masked_fill_(j[None, None, None, None, :] > last[:, None, None, :, None], float("-inf"))
    top = sc.amax(-1, keepdim=True).clamp(min=-3.0e38)
    w = sc.sub_(top).exp_()
    total = w.sum(-1, keepdim=True)
    o = torch.matmul(w.view(n, n_kv, -1, length), v).view(n, n_kv, h // n_kv, m, d) / total.clamp(min=1e-38)
    out = torch.cat([s["out"], torch.zeros_like(q[:1])])
    out[at] = o.permute(0, 3, 1, 2, 4).reshape(n, m, h, d).to(q.dtype)
    return out[:-1]


def _sample(s):
    c = s["case"]
    lg = s["logits"]
    if own:
        _, be = _be()
        be.sample_logits_dev(lg.shape[0], lg.shape[1], c["dt"], lg.data_ptr(), lg.stride(0), s["temp"].data_ptr(), s["top_k"].data_ptr(),
                             s["top_p"].data_ptr(), s["min_p"].data_ptr(), s["u"].data_ptr(), s["out"].data_ptr(), _stream())
        return s["out"]
    v = lg.shape[1]
    x, at = torch.sort(lg.double(), dim=-1, descending=True, stable=True)  # ties: the lowest index first
    temp = s["temp"].double()[:, None]
    w = torch.exp((x - x[:, :1]) / temp.clamp(min=1e-30))
    rank = torch.arange(v, device=lg.device)[None, :]
    k = s["top_k"].long()[:, None]
    w = torch.where((k <= 0) | (rank < k), w, 0.0)
    run_sum = torch.cumsum(w, -1)
    p = s["top_p"].double()[:, None]
    w = torch.where((p >= 1) | (run_sum - w < p * run_sum[:, -1:]) | (rank == 0), w, 0.0)
    w = torch.where(w >= s["min_p"].double()[:, None].clamp(max=1), w, 0.0)
    w = torch.zeros_like(w).scatter_(1, at, w)
    run_sum = torch.cumsum(w, -1)
    got = (run_sum <= s["u"].double()[:, None] * run_sum[:, -1:]).sum(-1).clamp(max=v - 1)
    return torch.where(s["temp"] > 0, got, at[:, 0]).to(torch.int32)


_RUN = {"plan": _plan, "store": _store, "attend": _attend, "sample": _sample}


# ---------------------------------------------------------------- 64 bits

def exact(case, seed):
    """The definition in 64 bits; the plan and the tokens are whole numbers."""
    op = case["op"]
    if op in ("plan", "sample"):
        return None
    s = prepare(case, seed)
    if op == "store":
        pool = torch.zeros(s["pool"].shape, dtype=torch.float64, device="cuda").transpose(1, 2).reshape(-1, 2, case["n_kv"], case["d"])
        live = s["slots"] >= 0
        at = s["slots"][live].long()
        pool[at, 0] = s["k"][live].double()
        pool[at, 1] = s["v"][live].double()
        return pool.view(case["pages"], case["page"], 2, case["n_kv"], case["d"]).transpose(1, 2)
    q, pool, p = s["q"], s["pool"], case["page"]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    cu, kv, group = s["cu"].tolist(), s["kv"].tolist(), case["n_head"] // case["n_kv"]
    for r in range(case["n_req"]):
        a, b, n = cu[r], cu[r + 1], kv[r]
        if b == a or n == 0:
            continue
        rows = pool[s["table"][r, : -(-n // p)].long()]
        for h in range(case["n_kv"]):
            k = rows[:, 0, :, h].reshape(-1, case["d"])[:n].double()
            v = rows[:, 1, :, h].reshape(-1, case["d"])[:n].double()
            for t in range(a, b, 1024):
                e = min(b, t + 1024)
                at = torch.arange(t, e, device="cuda") - b + n
                for g in range(h * group, (h + 1) * group):
                    x = q[t:e, g].double() @ k.T * s["scale"]
                    if case["causal"]:
                        x = torch.where(torch.arange(n, device="cuda")[None, :] <= at[:, None], x, -math.inf)
                    out[t:e, g] = torch.softmax(x, -1) @ v
    return out
