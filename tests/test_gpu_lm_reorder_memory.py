"""reorder_states where states and results lie in one memory: what is told apart, and what is refused."""
import random

import pytest
import torch

from spiky_amd import reorder_states

pytestmark = pytest.mark.gpu


def chosen(x, parents):
    return x[torch.arange(x.shape[0], device=x.device)[:, None], parents.long()].clone()


def test_used_positions_of_keys_and_values(cuda_device):
    """Keys and values of one cache whose runs lie as far apart as those of the other."""
    parents = torch.tensor([[0, 0, 1], [2, 1, 1]], device=cuda_device)
    for shape, used in (((2, 3, 2, 5, 40, 9), 17), ((2, 3, 2, 1, 40, 9), 39), ((2, 3, 2, 5, 7, 1), 1)):
        cache = torch.randn(*shape, device=cuda_device)
        whole = cache.clone()
        states = [cache[:, :, i, :, :used] for i in range(2)]
        for i, x in enumerate(states):
            whole[:, :, i, :, :used] = chosen(x, parents)
        reorder_states(states, parents, out=states)
        assert torch.equal(cache, whole)


def test_many_layers_of_one_cache(cuda_device):
    """Every layer's keys and values inside each beam."""
    cache = torch.randn(2, 4, 24, 2, 3, 20, 8, device=cuda_device).to(torch.bfloat16)
    parents = torch.tensor([[3, 0, 0, 1], [1, 1, 2, 3]], device=cuda_device)
    states = [cache[:, :, layer, i, :, :11] for layer in range(24) for i in range(2)]
    whole = cache.clone()
    whole[..., :11, :] = chosen(cache, parents)[..., :11, :]
    reorder_states(states, parents, out=states)
    assert torch.equal(cache, whole)


def layout(rng, counts, width):
    """Strides under which no byte is in it twice, and the bytes that it spans."""
    strides, span = [0] * 3, width
    for k in rng.sample(range(3), 3):
        strides[k] = span + rng.choice([0, 0, 5, width, 4 * width, 8 * width])
        span += strides[k] * (counts[k] - 1)
    return strides, span


def two_layouts(rng):
    """[(shape, strides, offset)] of two states of one memory, and whether they have a byte in common."""
    counts, widths = [rng.randint(1, 4) for _ in range(3)], [rng.choice([1, 2, 3, 16, 20]) for _ in range(2)]
    if rng.random() < 0.6:
        widths[1] = widths[0]
    alike = rng.random() < 0.7
    runs = rng.randint(1, counts[2] if alike else 4)
    first, span = layout(rng, counts, max(widths))
    second = first if alike else layout(rng, [*counts[:2], runs], widths[1])[0]
    at = [0, rng.randint(0, span + 3)]
    if rng.random() < 0.3:
        at.reverse()
    shapes = [(*counts, widths[0]), (*counts[:2], runs, widths[1])]
    places = [(shape, (*strides, 1), o) for shape, strides, o in zip(shapes, (first, second), at)]
    index = torch.arange(20000)
    sets = [set(index.as_strided(*p).flatten().tolist()) for p in places]
    assert all(len(s) == torch.Size(shape).numel() for s, shape in zip(sets, shapes))
    return places, bool(sets[0] & sets[1])


def test_any_two_layouts(cuda_device):
    """Refused where two states share a byte, and only there."""
    rng, found = random.Random(11), []
    for turn in range(300):
        places, shared = two_layouts(rng)
        found.append(shared)
        (searches, beams), gen = places[0][0][:2], torch.Generator().manual_seed(turn)
        base = torch.randint(0, 256, (20000,), generator=gen, dtype=torch.uint8)
        parents = torch.randint(0, beams, (searches, beams), generator=gen)
        there = base.to(cuda_device)
        states = [there.as_strided(*p) for p in places]
        if shared:
            with pytest.raises(ValueError, match="share no memory"):
                reorder_states(states, parents.to(cuda_device), out=states)
            continue
        reorder_states(states, parents.to(cuda_device), out=states)
        want = base.clone()
        for p in places:
            want.as_strided(*p).copy_(chosen(base.as_strided(*p), parents))
        assert torch.equal(there.cpu(), want), (turn, places)
    assert 60 <= sum(found) <= 240


@pytest.mark.parametrize("flip", [False, True])
def test_runs_that_do_not_nest(cuda_device, flip):
    """Positions in use of a cache into rows with a gap behind each, and the other way."""
    parents = torch.tensor([[0, 0, 1], [2, 1, 1]], device=cuda_device)
    cache, rows = torch.randn(2, 3, 5, 40, 9, device=cuda_device), torch.randn(2, 3, 5, 16, 12, device=cuda_device)
    x, out = (rows[..., :9], cache[:, :, :, :16]) if flip else (cache[:, :, :, :16], rows[..., :9])
    kept, before, want = (cache if flip else rows).clone(), x.clone(), chosen(x, parents)
    (kept[:, :, :, :16] if flip else kept[..., :9]).copy_(want)
    assert reorder_states([x], parents, out=[out])[0] is out
    assert torch.equal(cache if flip else rows, kept) and torch.equal(x, before)


@pytest.mark.parametrize("beams,n", [(4, 4), (8, 8), (16, 16), (31, 31), (64, 64), (64, 100), (7, 130)])
def test_results_past_the_last_cache(cuda_device, beams, n):
    """More than 512 MiB of results, runs that end inside 16 bytes, some beams that stay and parents that there are none of."""
    width = ((600 << 20) // (2 * n * 3) & ~15) + 13
    gen = torch.Generator(cuda_device).manual_seed(n)
    x = torch.randint(0, 256, (2, beams, 3, width), generator=gen, device=cuda_device, dtype=torch.uint8)
    parents = torch.randint(0, beams, (2, n), generator=gen, device=cuda_device)
    parents[0, :min(beams, n) // 2] = torch.arange(min(beams, n) // 2, device=cuda_device)
    parents[1, n - 1] = -1
    want = torch.where((parents >= 0)[:, :, None, None], chosen(x, parents.clamp_min(0)), 0)
    assert torch.equal(reorder_states(x, parents), want)
    if n == beams:
        reorder_states(x, parents, out=x)
        assert torch.equal(x, want)


def test_every_other_value_in_two_groupings(cuda_device):
    """One state's values lie 2 apart, the other's 4, between them: told apart without going through all."""
    base = torch.randint(0, 256, (2, 3, 1 << 18, 2), device=cuda_device, dtype=torch.uint8)
    states = [base[..., 0], base.view(2, 3, 1 << 17, 4)[..., 1]]
    parents = torch.tensor([[0, 0, 1], [2, 1, 1]], device=cuda_device)
    want = base.clone()
    want[..., 0] = chosen(states[0], parents)
    want.view(2, 3, 1 << 17, 4)[..., 1] = chosen(states[1], parents)
    reorder_states(states, parents, out=states)
    assert torch.equal(base, want)
