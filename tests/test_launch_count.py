"""Kernels that a call of the paged attention says it launched."""
import types

import pytest
import torch


@pytest.mark.parametrize("groups,q_lens,launches", [([(4, 0)], 1, 2), ([(3, 0)], 100, 2), ([(2, 0)], [1, 100], 3),
                                                    ([(100, 6400)], 1, 3), ([(2, 0)], 0, 0), ([], 1, 0)])
def test_paged_attention(groups, q_lens, launches, monkeypatch):
    from rs_nanogpt_b200.ops import _ext, paged
    fake = _ext._Counted(types.SimpleNamespace(paged_attention=lambda *a: None))
    monkeypatch.setattr(paged, "ext", lambda: fake)
    plan = paged.PrefixPlan(groups, q_lens, n_head=2, n_kv_head=2, head_dim=64, page=64, table_width=128, device="cpu")
    before = _ext.launch_count()
    paged.attention(torch.zeros(plan.rows, 2, 64), None, None, None, None, plan)
    assert _ext.launch_count() - before == launches
