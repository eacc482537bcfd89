"""A sparse prefill whose rotated keys and values go into the pages, then tokens served from them, on the GPU."""
from __future__ import annotations

import pytest
import torch

import fftsparse_amd as fa
from tests.test_gpu_serving_split import check

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, I32 = torch.bfloat16, torch.int32


@pytest.mark.parametrize("hnd", [False, True])
def test_tokens_after_a_sparse_prefill(hnd):
    L, Hq, Hk, D, ps, pages = 1700, 8, 2, 128, 64, 60
    g = torch.Generator().manual_seed(0)
    new = lambda T: [torch.randn(T, h, D, generator=g).to(BF).to(DEV) for h in (Hq, Hk, Hk)]   # noqa: E731
    inv, _ = fa.rope_frequencies(D, base=500000.0)
    angle = torch.arange(L, device=DEV)[:, None] * inv
    cos, sin = (torch.cat([f(angle)] * 2, -1).to(BF) for f in (torch.cos, torch.sin))
    shape = (pages, Hk, ps, D) if hnd else (pages, ps, Hk, D)
    k_cache, v_cache = (torch.full(shape, float("nan"), dtype=BF, device=DEV) for _ in range(2))
    if hnd:
        k_cache, v_cache = k_cache.transpose(1, 2), v_cache.transpose(1, 2)
    table = torch.full((2, 40), -1, dtype=I32, device=DEV)
    free = torch.randperm(pages, generator=g).to(I32).to(DEV)
    ints = lambda *x: torch.tensor(x, dtype=I32, device=DEV)              # noqa: E731
    lens, count = ints(0, 0), ints(pages)

    q, k, v = (x.transpose(0, 1)[None] for x in new(L))                    # [1, H, L, D] views
    q_rot, k_rot, q_b, k_b = fa.rope_pool(q, k, cos, sin, block_size=128)
    sel = fa.select_blocks(q_rot, k_rot, block_size=128, corr_threshold=0.9, pooled=(q_b, k_b))
    out = fa.block_sparse_attention(q_rot, k_rot, v, sel.blk_cnt, sel.blk_bits)
    assert out.shape == (1, L, Hq, D)
    plan = fa.plan_step(table, lens, ints(0, L), free, count, page_size=ps, num_tokens=L)
    k_cache[plan.slots // ps, plan.slots % ps] = k_rot[0].transpose(0, 1)
    v_cache[plan.slots // ps, plan.slots % ps] = v[0].transpose(0, 1)

    keys, values = k_rot[0].transpose(0, 1), v[0].transpose(0, 1)
    for T in (1, 5):
        lens, count = plan.seq_lens, plan.free_count
        q, k, v = new(T)
        plan = fa.plan_step(table, lens, ints(0, T), free, count, page_size=ps, num_tokens=T)
        r, rk = fa.rope(q, k, plan.positions, inv)
        assert torch.equal(fa.rope_cache(q, k, v, plan.positions, plan.slots, k_cache, v_cache, inv), r)
        first = len(keys)
        keys, values = torch.cat([keys, rk]), torch.cat([values, v])
        got = fa.paged_attention(r, k_cache, v_cache, table, plan.cu_lens, plan.seq_lens, max_new=T)
        check(got, r.cpu(), keys.cpu(), values.cpu(), first, None, 0, T)
    assert plan.seq_lens.tolist() == [0, L + 6] and int(plan.lacking) == 0
