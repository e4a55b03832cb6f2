"""Front-end calls around drafted trees whose parts do not fit each other: refused on the host, before a device indexes past an end."""
from __future__ import annotations

import pytest
import torch

from vllm_webgpu_amd.v1.kv_cache import PagedKVCache
from vllm_webgpu_amd.v1.sample.metadata import SamplingMetadata
from vllm_webgpu_amd.v1.sample.tree_sampler import DraftTree, TreeSampler

CPU = torch.device("cpu")


@pytest.mark.parametrize("name", ["temperature", "top_k", "top_p", "min_p"])
@pytest.mark.parametrize("count", [1, 2, 4])
def test_settings_of_another_count_of_requests(name, count):
    tree = DraftTree.make([[-1, 0], [-1], [-1, 0, 0]], CPU)
    fine = dict(temperature=torch.ones(3), top_k=None, top_p=None)
    m = SamplingMetadata(**{**fine, **({} if name == "min_p" else {name: torch.ones(count)})}, all_greedy=False, all_random=True, generators={},
                         max_num_logprobs=None, no_penalties=True, prompt_token_ids=None, frequency_penalties=None, presence_penalties=None,
                         repetition_penalties=None, output_token_ids=[])
    if name == "min_p":
        m.min_p = torch.ones(count)
    with pytest.raises(ValueError, match=name):
        TreeSampler()(tree, torch.zeros(6, dtype=torch.int32), torch.zeros((6, 20)), m)


@pytest.mark.parametrize("tables,contexts", [(2, 3), (3, 2), (4, 3), (3, 4), (2, 2)])
def test_tables_and_contexts_of_another_count_of_requests(tables, contexts):
    c = PagedKVCache(1, 10, 1, 64, page_size=16, device="cpu")
    for i in range(4):
        c.reserve(str(i), 20)
    tree = DraftTree.make([[-1, 0], [-1], [-1, 0, 0]], CPU)
    table = c.block_table([str(i) for i in range(4)])
    with pytest.raises(ValueError):
        c.slots(table[:tables], torch.zeros(contexts, dtype=torch.int32), tree)
    assert c.slots(table[:3], torch.zeros(3, dtype=torch.int32), tree).shape == (6,)
