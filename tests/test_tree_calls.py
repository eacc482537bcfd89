"""CPU tests of calls of the tree operators that cannot be taken: refused before any launch, at the C ABI and in Python."""
from __future__ import annotations

import ctypes

import pytest
import torch

import fftsparse_amd as fa
from fftsparse_amd import _lib
from oracle import paged, tree
from tests.test_serving_host import BF, I32, _paged, _rc
from tests.test_tree_host import _eight

PAGE = 16 * 2 * 128 * 2                                    # bytes of a page of 16 tokens, 2 heads of 128, 16 bits
SIZE = 8 * PAGE                                            # of a cache
AT = 1 << 30


def _move(k, v, **kw):
    """A move in caches at the given addresses (lists: a sequence of layers; numbers: layers by a stride)."""
    args = dict(block_table=16, t_sb=4, cu_lens=16, seq_lens=16, kept=16, layers=2, B=2, T=3, Hk=2, D=128, P=4, page_size=16,
                elem_bytes=2, num_pages=8, k_sp=4096, k_ss=256, k_sh=128, v_sp=4096, v_ss=256, v_sh=128)
    if isinstance(k, list):
        arrays = [(ctypes.c_void_p * len(x))(*x) for x in (k, v)]
        args.update(k_caches=arrays[0], v_caches=arrays[1], layers=len(k))
    else:
        args.update(k_cache=k, v_cache=v, k_sl=SIZE // 2, v_sl=SIZE // 2)
    return _lib.CacheMoveArgs(**{**args, **kw})


@pytest.mark.parametrize("k,v,kw", [
    ([AT, AT], [AT + SIZE, AT + 2 * SIZE], {}),                                        # layers of one cache of keys
    ([AT, AT + SIZE], [AT + 2 * SIZE, AT + 2 * SIZE], {}),                             # and of values
    ([AT, AT + SIZE, AT], [AT + 2 * SIZE, AT + 3 * SIZE, AT + 2 * SIZE], {}),          # both, not side by side
    ([AT], [AT], {}),                                                                  # keys and values in one
    ([AT + SIZE, AT], [AT + 2 * SIZE, AT + SIZE], {}),
    ([AT, AT + SIZE // 2], [AT + 2 * SIZE, AT + 3 * SIZE], {}),                        # caches that overlap by half
    ([AT], [AT + 7 * PAGE], {}),                                                       # by a page
    ([AT], [AT + SIZE - 256], {}),                                                     # by the last token's last head
    ([AT], [AT + 256], {}),
    ([AT], [AT + SIZE - 256], dict(v_ss=128, v_sh=16 * 128)),                          # of different layouts
    ([AT + i * 100 * SIZE for i in range(70)] + [AT], [AT + (i * 100 + 1) * SIZE for i in range(71)], {}),   # two launches
    # 40 layers side by side in each page, or in each token, one of them twice, or values a head too early
    ([AT + i % 39 * 2 * PAGE for i in range(40)], [AT + (2 * i + 1) * PAGE for i in range(40)], dict(k_sp=40 * PAGE, v_sp=40 * PAGE)),
    ([AT + 2 * i * PAGE for i in range(40)], [AT + (2 * i + 1) * PAGE - 256 for i in range(40)], dict(k_sp=40 * PAGE, v_sp=40 * PAGE)),
    ([AT + 1024 * i for i in range(40)], [AT + 1024 * (i % 39) + 512 for i in range(40)],
     dict(k_sp=40 * PAGE, v_sp=40 * PAGE, k_ss=20480, v_ss=20480)),
    ([AT + 1024 * i for i in range(40)], [AT + 1024 * i + 256 for i in range(40)],
     dict(k_sp=40 * PAGE, v_sp=40 * PAGE, k_ss=20480, v_ss=20480)),
    ([AT, AT + 256], [AT + SIZE, AT + 2 * SIZE], dict(k_sp=-4096)),                    # backwards
    (AT, AT, {}),
    (AT, AT + SIZE, {}),                                                               # the values are the second layer's keys
    (AT, AT + 2 * SIZE, dict(k_sl=0)),                                                 # layers by a stride that is none,
    (AT, AT + 2 * SIZE, dict(v_sl=0)),
    (AT, AT + 4 * SIZE, dict(k_sl=2048)),                                              # or too short
    (AT, AT + 4 * SIZE, dict(v_sl=4096 * 7)),
    (AT, AT + 256, dict(k_sp=8192, k_ss=512, k_sh=128, v_sp=8192, v_ss=512, v_sh=128, k_sl=SIZE, v_sl=SIZE)),
])
def test_caches_of_a_move_that_share_storage_are_refused(k, v, kw):
    """Each cache is moved by workgroups of its own: one that is named twice would be moved twice."""
    got, said = _rc("fs_cache_move", _move(k, v, **kw))
    assert (got, "share storage" in said) == (-1, True), (got, said)


def test_plan_tree_refuses_windows():
    p, cu, lens = torch.zeros(6, dtype=I32), torch.zeros(4, dtype=I32), torch.zeros(3, dtype=I32)
    for text, kw in [("on the GPU", dict(window=5, sinks=2)), ("on the GPU", dict(window=2 ** 31 - 1, sinks=2 ** 31 - 1)),
                     ("window", dict(window=0)), ("window", dict(window=2 ** 31)), ("sinks", dict(window=5, sinks=-1))]:
        with pytest.raises(ValueError, match=text):
            fa.plan_tree(p, cu, lens, max_new=4, **kw)
    args = _lib.TreePlanArgs(parents=16, cu_lens=16, seq_lens=16, B=2, T=3, words=1, positions=16, mask=16)
    for change in (dict(window=-1), dict(window=1, sinks=-1)):
        got, said = _rc("fs_tree_plan", args, **change)
        assert (got, "must not be negative" in said) == (-1, True), said


@pytest.mark.parametrize("window,sinks", [(1, 0), (3, 0), (3, 22), (5, 23), (4, 100), (8, 0), (25, 2), (None, 0)])
def test_the_oracle_of_a_chain_is_that_of_paged_attention_under_any_window(window, sinks):
    """Windows shorter than the chain too: the new tokens that it hides are hidden."""
    g = torch.Generator().manual_seed(0)
    q, k, v = torch.randn(9, 4, 16, generator=g), *(torch.randn(30, 2, 16, generator=g) for _ in range(2))
    pos, mask = tree.plan([-1, *range(8)], [0, 9], [30], 1, window, sinks)
    sees = torch.tensor([[m[0] >> j & 1 for j in range(9)] for m in mask], dtype=torch.bool)
    a = tree.attend(q, k, v, 9, sees, window, sinks, pos=pos)[0]
    b = paged.attend(q, k, v, 21, window, sinks)[0]
    assert torch.allclose(a, b, atol=1e-12)


def test_outputs_that_share_storage_are_refused(monkeypatch):
    """With each other, or with what the kernels still read when they are written (the check that these tensors are on a GPU is
    left out, so that the next one is reached; nothing is launched)."""
    monkeypatch.setattr(_lib, "same_device", lambda *tensors: tensors[0].device)
    monkeypatch.setattr(_lib, "call", lambda name, *rest: pytest.fail(f"{name} was launched"))
    p, cu, lens, x = torch.zeros(6, dtype=I32), torch.zeros(4, dtype=I32), torch.zeros(3, dtype=I32), torch.zeros(6, dtype=torch.int64)
    buf = torch.zeros(64, dtype=torch.int64)
    half = buf.view(I32)
    for out, text in [(fa.TreePlan(half[5:11], buf[:6].view(6, 1)), "each other"), (fa.TreePlan(half[:6], buf[:6].view(6, 1)), "each other"),
                      (fa.TreePlan(p, buf[:6].view(6, 1)), "an input")]:
        with pytest.raises(ValueError, match=text):
            fa.plan_tree(p, cu, lens, max_new=4, out=out)
    small = torch.zeros(3, dtype=I32)
    for out, text in [(fa.Accepted(half[:6], small, small, buf[20:23]), "each other"),
                      (fa.Accepted(half[:6], half[5:8], small, buf[20:23]), "each other"),
                      (fa.Accepted(half[:6], small, half[42:45], buf[20:23]), "each other"),
                      (fa.Accepted(half[:6], small, half[8:11], x[:3]), "an input")]:
        with pytest.raises(ValueError, match=text):
            fa.accept_tree(p, x, x.clone(), cu, max_new=4, out=out)
    a = _paged()
    rows = torch.zeros(4096 + 6 * 2048, dtype=torch.uint8)                  # out's rows in 8 bytes of each 2048
    out = rows.view(BF)[:6 * 1024].view(6, 1024)[:, :512].view(6, 4, 128)
    inside = rows[1024:1024 + 48].view(torch.int64).view(6, 1)              # behind a row, within the tensor's span
    for kw in [dict(mask=torch.zeros(6 * 128, dtype=torch.int64)), dict(mask=inside),
               dict(mask=torch.zeros(6, 1, dtype=torch.int64), window=3, positions=rows[2048:2048 + 24].view(I32))]:
        if kw["mask"].dim() == 1:
            whole = kw["mask"]
            kw["mask"], o = whole[:6].view(6, 1), whole.view(BF)[:6 * 512].view(6, 4, 128)
        else:
            o = out
        with pytest.raises(ValueError, match="an input"):
            fa.tree_attention(**a, **kw, out=o)
    e = _eight()
    scale = torch.zeros(6 * 256)
    with pytest.raises(ValueError, match="an input"):
        fa.paged_attention(**{**e, "k_scale": scale[:2]}, out=scale.view(BF)[:6 * 512].view(6, 4, 128))
