"""The gradient of large tables of relative_attention: buckets times offsets from 2^28 on, and as many buckets as it takes."""
import pytest
import torch

from tests.test_ops_relative_attention_gpu import check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_a_bucket_for_every_offset(gpu_device, dtype):
    """In the map's order, in one of its own, clipped far from the query, and with offsets that have none."""
    t, _, mask, start, do = make(gpu_device, 2, 3, (65, 65), 16, dtype, queries=20, start=2100, masked=True, seed=30)
    g = torch.Generator().manual_seed(31)
    n = 129 * 129
    assert n * n >= 1 << 28
    t[3] = torch.randn((n, 3), generator=g).to(dtype).to(gpu_device)
    every = torch.arange(n, dtype=torch.int32).reshape(129, 129)
    far = (torch.arange(129) - 64).clamp(-10, 10) + 10
    holes = every.clone()
    holes[::3, ::2] = -1
    holes[5, 5] = n
    holes[6, 6], holes[7, 7] = -2 ** 31, 2 ** 31 - 1
    for buckets in (every, every.flatten()[torch.randperm(n, generator=g)].reshape(129, 129),
                    (n - 1 - far[:, None] * 21 - far[None]).int(), holes):
        check(t, buckets.contiguous().to(gpu_device), mask, start, do)


def test_the_largest_table(gpu_device):
    """2^24 buckets, of which a small grid has a few: the others' gradients are zero."""
    t, _, mask, start, do = make(gpu_device, 1, 1, (5, 6), 8, torch.float32, seed=32)
    g = torch.Generator().manual_seed(33)
    t[3] = torch.randn((1 << 24, 1), generator=g).to(gpu_device)
    buckets = torch.randint(0, 1 << 24, (9, 11), generator=g, dtype=torch.int32)
    buckets[0, 0], buckets[4, 5], buckets[8, 10] = 0, (1 << 24) - 1, 1 << 20
    buckets = buckets.to(gpu_device)
    _, grads = check(t, buckets, mask, start, do)
    rest = torch.ones(1 << 24, dtype=torch.bool, device=gpu_device)
    rest[buckets.flatten().long()] = False
    assert (grads[3][rest] == 0).all() and grads[3][(1 << 24) - 1] != 0
