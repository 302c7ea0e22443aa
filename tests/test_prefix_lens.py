"""The lengths that a shared-prefix plan keeps on the device behind its words."""

from __future__ import annotations

import pytest
import torch

from cacheslide_b200.prefix import SharedPrefixAttention


@pytest.mark.parametrize("query,suffix", [([1], [1]), ([3, 0, 17], [9, 0, 17]), ([0], [0]), ([], []),
                                          ([1] * 500, list(range(1, 501))),
                                          ([5, 2], [2 ** 20, 3])])
def test_lengths_lie_behind_the_words(query, suffix):
    plan = SharedPrefixAttention(8, 2, 128, torch.bfloat16, "cpu", query_lens=query,
                                 suffix_lens=suffix, prefix_lens=[40])
    lens = plan.device_lens
    assert lens.dtype is torch.int32 and lens.tolist() == [query, suffix]
    assert plan.words.numel() == plan.info.words
    assert lens.data_ptr() == plan.words.data_ptr() + 4 * plan.info.words or not plan.tokens
    # the same plan again has the same words: nothing of the lengths in them
    again = SharedPrefixAttention(8, 2, 128, torch.bfloat16, "cpu", query_lens=query,
                                  suffix_lens=suffix, prefix_lens=[40])
    assert torch.equal(again.words, plan.words) and torch.equal(again.device_lens, lens)
