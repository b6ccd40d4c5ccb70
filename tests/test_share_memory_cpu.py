"""Whether views of one buffer share memory, against the sets of their bytes."""
import random

import pytest
import torch

from rdkv_b200._lib import share_memory


def places(t):
    at = torch.zeros((), dtype=torch.int64)
    for n, st in zip(t.shape, t.stride()):
        at = at[..., None] + torch.arange(n) * st
    first = (at.reshape(-1) * t.element_size() + t.data_ptr()).tolist()
    return {x + e for x in first for e in range(t.element_size())}


def view(rng, buf):
    shape = [rng.choice([0, 1, 1, 2, 3, 5, 8]) for _ in range(rng.choice([1, 2, 3]))] + [rng.choice([1, 4, 6])]
    stride, at = [1], shape[-1]
    for n in reversed(shape[:-1]):
        step = rng.choice([at, at, at + 1, 2 * at, at + 4, 7, 0])
        stride.append(step)
        at = max(at, step * n)
    stride = stride[::-1]
    room = buf.numel() - 1 - sum((n - 1) * st for n, st in zip(shape, stride))
    return buf.as_strided(shape, stride, rng.randint(0, min(room, rng.choice([3, 40, room])))) if room >= 0 else buf[:5]


@pytest.mark.parametrize("seed", range(40))
def test_share_memory(seed):
    rng = random.Random(seed)
    raw = torch.zeros(2400, dtype=torch.uint8)
    for _ in range(100):
        a, b = (view(rng, raw.view(rng.choice([torch.float16, torch.float32, torch.uint8]))) for _ in range(2))
        assert share_memory(a, b) == bool(places(a) & places(b)), (a.shape, a.stride(), b.shape, b.stride())


def test_views_of_a_fused_projection():
    both = torch.zeros(50, 12, 136)
    q, k, v = both[:, :6, :128], both[:, 6:9, :128], both[:, 9:, :128]
    assert not share_memory(q, k) and not share_memory(k, v) and not share_memory(v, q) and share_memory(q, q)
    assert not share_memory(both[..., :128], both[..., 128:]) and share_memory(q[:-1], q[1:]) and not share_memory(q[:25], q[25:])
    assert not share_memory(q[::2], q[1::2]) and share_memory(q[::2], q[::3]) and not share_memory(q[:0], q)
