"""Copies of more pages than one launch holds (2^24 blocks of 256 threads less one)."""
import pytest
import torch

from vortex_amd import kv_copy_pages

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_more_small_pages_than_a_launch_holds():
    n = (1 << 24) + 1000
    pools = torch.zeros(1, 2 * n, 16, dtype=torch.uint8, device=DEV)
    at = torch.arange(n, dtype=torch.int32, device=DEV)
    pools[0, :n].view(torch.int32).copy_(at[:, None] * torch.tensor([1, 3, 5, 7], dtype=torch.int32, device=DEV))
    kv_copy_pages(pools, at, at + n)
    assert torch.equal(pools[0, n:], pools[0, :n])


def test_more_pieces_than_a_launch_holds():
    # pages of four pieces, most pairs name none; those at the launches' ends do
    size, P, most = 3 * 4096 + 7, 40, ((1 << 24) - 1) // 4
    n = 2 * most + 5
    pools = torch.randint(0, 255, (3, P, size), dtype=torch.uint8, device=DEV)
    src, dst = (torch.full((n,), -1, dtype=torch.int32, device=DEV) for _ in range(2))
    ends = [0, 1, most - 1, most, most + 1, 2 * most - 1, 2 * most, n - 1]
    src[ends] = torch.arange(len(ends), dtype=torch.int32, device=DEV)
    dst[ends] = torch.arange(20, 20 + len(ends), dtype=torch.int32, device=DEV)
    want = pools.clone()
    want[:, 20:20 + len(ends)] = pools[:, :len(ends)]
    kv_copy_pages(pools, src, dst)
    assert torch.equal(pools, want)
