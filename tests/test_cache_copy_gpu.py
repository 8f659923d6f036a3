"""Copies of cache pages and state slots: bit for bit, and nothing beside them."""

import pytest
import torch

from freetoken_b200.errors import KernelError
from freetoken_b200.kernels import ops

DEV = "cuda:0"


def noise(shape, dtype, seed):
    """Bits of every kind, NaN among them."""
    g = torch.Generator().manual_seed(seed)
    size = torch.tensor([], dtype=dtype).element_size()
    raw = torch.randint(0, 256, (*shape, size), generator=g, dtype=torch.uint8)
    return raw.view(dtype).reshape(shape)


def bits(t):
    return t.cpu().contiguous().view(torch.uint8)


def plain(t, pairs):
    new = t.clone()
    for pair in pairs:
        if len(pair) == 2:
            new[:, pair[1]] = t[:, pair[0]]
        else:
            new[:, pair[1], :, :pair[2]] = t[:, pair[0], :, :pair[2]]
    return new


def on_device(pairs, ints):
    return torch.tensor(pairs, dtype=torch.int32, device=DEV).reshape(-1, ints)


@pytest.mark.gpu
@pytest.mark.parametrize("shape,dtype", [
    ((1, 9, 1, 1, 16), torch.bfloat16), ((3, 9, 8, 16, 128), torch.bfloat16), ((2, 9, 4, 16, 64), torch.float32), ((2, 9, 2, 7, 48), torch.bfloat16),
    ((5, 9, 3, 4, 9), torch.bfloat16), ((1, 9, 1, 5, 3), torch.uint8), ((2, 9, 1, 64, 256), torch.float32),
])
def test_pages(shape, dtype):
    P = shape[3]
    slabs = [noise(shape, dtype, s) for s in (1, 2)] + [noise((shape[0] + 1, shape[1], 2, P, shape[4]), dtype, 3)]
    pairs = [(2, 5, 1), (2, 6, P), (2, 1, max(1, P // 2)), (4, 3, P - 1), (7, 7, P), (8, 0, P + 5)]
    here = [t.to(DEV) for t in slabs]
    ops.copy_pages(here, on_device(pairs, 3))
    for t, h in zip(slabs, here):
        assert torch.equal(bits(h), bits(plain(t, pairs)))


@pytest.mark.gpu
@pytest.mark.parametrize("tail", [(3,), (16, 64, 64), (2, 5), (), (1000,), (3, 33000)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_slots(tail, dtype):
    tensors = [noise((2, 6, *tail), dtype, 1), noise((4, 6, 7), dtype, 2)]
    pairs = [(1, 2), (1, 3), (4, 5)]
    here = [t.to(DEV) for t in tensors]
    ops.copy_slots(here, on_device(pairs, 2))
    for t, h in zip(tensors, here):
        assert torch.equal(bits(h), bits(plain(t, pairs)))


@pytest.mark.gpu
def test_more_tensors_than_one_launch_takes_and_views_that_start_anywhere():
    whole = [noise((2, 5, 1, 4, 6), torch.bfloat16, s) for s in range(37)]
    whole = [t if i % 3 else torch.cat([t.reshape(-1)[:1], t.reshape(-1)]) for i, t in enumerate(whole)]  # (2 bytes past a boundary)
    here = [t.to(DEV) for t in whole]
    views = [h if h.dim() == 5 else h[1:].view(2, 5, 1, 4, 6) for h in here]
    refs = [plain(h.cpu(), [(1, 4, 3)]) for h in views]
    before = ops.launch_count()
    ops.copy_pages(views, on_device([(1, 4, 3)], 3))
    assert ops.launch_count() - before == 3
    for h, ref in zip(views, refs):
        assert torch.equal(bits(h), bits(ref))
    for h, t in zip(here, whole):
        if h.dim() == 1:
            assert torch.equal(bits(h[:1]), bits(t[:1]))


@pytest.mark.gpu
def test_pairs_outside_the_tensor_do_nothing():
    t = noise((2, 5, 2, 4, 8), torch.bfloat16, 1)
    here = t.to(DEV)
    ops.copy_pages([here], on_device([(-1, 2, 4), (2, -1, 4), (5, 2, 4), (2, 5, 4), (2, 1 << 30, 4), (1, 2, 0), (1, 2, -3), (3, 3, 4)], 3))
    ops.copy_pages([here], on_device([], 3))
    ops.copy_slots([here], on_device([(0, 5), (7, 1), (-2, 1)], 2))
    assert torch.equal(bits(here), bits(t))


@pytest.mark.gpu
def test_a_slab_past_32_bit_offsets():
    """Entries behind 2^32 bytes and 2^31 elements."""
    slab = torch.zeros((3, 70000, 1, 16, 1024), dtype=torch.bfloat16, device=DEV)  # 6.9 GB
    slab[2, 69990] = 1.5
    slab[1, 69990] = 2.5
    ops.copy_pages([slab], on_device([(69990, 69999, 9)], 3))
    assert (slab[2, 69999, :, :9] == 1.5).all() and (slab[1, 69999, :, :9] == 2.5).all() and not slab[2, 69999, :, 9:].any()
    assert not slab[0].any() and not slab[2, :69990].any()


@pytest.mark.gpu
def test_captured_and_replayed_with_other_pairs():
    t = noise((2, 6, 2, 4, 64), torch.bfloat16, 1).to(DEV)
    start, pairs = t.clone(), on_device([(1, 2, 4)], 3)
    ops.copy_pages([t], pairs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.copy_pages([t], pairs)
    for pair in [(3, 5, 2), (0, 4, 4)]:
        t.copy_(start)
        pairs.copy_(torch.tensor([pair], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(bits(t), bits(plain(start, [pair])))


def test_refusals_without_a_gpu():
    slab, pairs = torch.zeros((1, 4, 1, 2, 8)), torch.zeros((1, 3), dtype=torch.int32)
    for slabs, p in [([slab], pairs), ([slab], pairs.long()), ([slab], pairs[0]), ([slab], pairs[:, :2]), ([slab[0]], pairs),
                     ([slab, torch.zeros((1, 5, 1, 2, 8))], pairs), ([slab, torch.zeros((1, 4, 1, 3, 8))], pairs), ([slab[:0]], pairs)]:
        with pytest.raises(KernelError):
            ops.copy_pages(slabs, p)
    for tensors, p in [([slab], pairs), ([slab[0, 0, 0, 0]], pairs[:, :2]), ([slab, torch.zeros(1, 5)], pairs[:, :2]), ([slab[:0]], pairs[:, :2])]:
        with pytest.raises(KernelError):
            ops.copy_slots(tensors, p)


@pytest.mark.gpu
def test_refusals():
    slab = torch.zeros((2, 4, 2, 4, 8), device=DEV)
    with pytest.raises(KernelError, match="contiguous"):
        ops.copy_pages([slab.transpose(2, 3)], on_device([(1, 2, 2)], 3))
    with pytest.raises(KernelError, match="device"):
        ops.copy_pages([slab], torch.zeros((1, 3), dtype=torch.int32))
