"""Pools that are views: a pool of one layer cut out of a tensor with the layers first is contiguous
whatever its stride between layers is, and only its own keys and values may be touched."""

from __future__ import annotations

import numpy as np
import pytest
import torch


def _one_layer(layers_first: torch.Tensor, layer: int) -> torch.Tensor:
    """(2, 1, blocks, heads, block size, d_head) of one layer of a (layers, 2, ...) tensor."""
    pool = layers_first[layer : layer + 1].transpose(0, 1)
    assert pool.is_contiguous() and pool.stride(1) != pool.stride(0)
    return pool


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_addresses_of_a_pool_go_by_its_sizes(dtype) -> None:
    from microserve_b200.cache import _pack_pool

    whole = torch.zeros((4, 2, 3, 2, 8, 6), dtype=dtype)
    for layer in range(4):
        pool = _one_layer(whole, layer)
        _, at = _pack_pool(pool, -1)
        assert at.tolist() == [pool[0, 0].data_ptr(), pool[1, 0].data_ptr()]
    several = torch.zeros((2, 5, 3, 2, 8, 6), dtype=dtype)
    _, at = _pack_pool(several, -1)
    assert at.tolist() == [several[i, l].data_ptr() for i in range(2) for l in range(5)]
    for empty in (torch.zeros((2, 0, 3, 2, 8, 6)), torch.zeros((2, 2, 0, 2, 8, 6))):
        assert len(_pack_pool(empty, -1)[1]) == 2 * empty.shape[1]


@pytest.mark.gpu
@pytest.mark.parametrize("layer", range(4))
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_copies_and_moves_in_one_layer_of_many(dtype, layer) -> None:
    from microserve_b200.cache import copy_blocks, move_tokens

    i32 = lambda a: torch.from_numpy(np.array(a, np.int32)).cuda()  # noqa: E731
    whole = torch.randn((4, 2, 6, 2, 8, 16), device="cuda").to(dtype)
    want = whole.clone()
    pool = _one_layer(whole, layer)
    copy_blocks(pool, i32([0, 5]), i32([1, 2]))
    want[layer, :, 1], want[layer, :, 2] = want[layer, :, 0].clone(), want[layer, :, 5].clone()
    assert torch.equal(whole, want)
    move_tokens(pool, i32([[8 * 3 + 1, 8 * 4 + 7]]), i32([[8 * 4 + 7, 8 * 5 + 2]]))
    want[layer, :, 5, :, 2] = want[layer, :, 4, :, 7]
    want[layer, :, 4, :, 7] = want[layer, :, 3, :, 1]
    assert torch.equal(whole, want)
