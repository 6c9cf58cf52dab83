"""CPU: the runs of decodes and chunks that the vLLM metadata of a mixed step
carries (the attention's choice of calls)."""

from types import SimpleNamespace

import pytest
import torch


@pytest.mark.parametrize("q_lens,want", [
    ([], []), ([1], [(0, 1, 0, True)]), ([5], [(0, 1, 0, False)]),
    ([1, 1, 1, 7, 0, 2], [(0, 3, 0, True), (3, 6, 3, False)]),
    ([0, 9, 1, 1], [(0, 2, 0, False), (2, 4, 9, True)]),
    ([1, 2, 1], [(0, 1, 0, True), (1, 2, 1, False), (2, 3, 3, True)])])
def test_query_runs(q_lens, want):
    from kessie_b200.kessie_attention import query_runs
    starts = [sum(q_lens[:i]) for i in range(len(q_lens) + 1)]
    assert [tuple(r) for r in query_runs(starts)] == want
    assert [tuple(r) for r in query_runs(starts, 2)] == (want if len(want) <= 2 else [])


def test_builder_adds_the_runs_to_flash_attentions_metadata(monkeypatch):
    from kessie_b200 import kessie_attention as A
    if not A.HAS_VLLM:
        pytest.skip("vLLM is not installed")
    cls = A.KeSSieAttentionBackend.get_builder_cls()
    parent = A.KeSSieAttentionBackend._get_original().get_builder_cls()
    assert issubclass(cls, parent)
    made = SimpleNamespace()
    monkeypatch.setattr(parent, "build", lambda self, *a: made)
    builder = object.__new__(cls)
    common = SimpleNamespace(query_start_loc_cpu=torch.tensor([0, 1, 2, 9], dtype=torch.int32), max_query_len=7)
    assert builder.build(0, common) is made
    assert made.query_runs == (A.QueryRun(0, 2, 0, True), A.QueryRun(2, 3, 2, False))
    del made.query_runs
    common.max_query_len = 1                                         # a decode step has no use for them
    assert builder.build(0, common_attn_metadata=common, fast_build=True) is made and not vars(made)
