"""reorder_states on the GPU against torch's indexing: values are moved, so results are equal."""
import pytest
import torch

from spiky_amd import reorder_states

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.uint8, torch.int64, torch.bool, torch.float64, torch.complex128]


def state(shape, dtype, device, seed=0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randint(0, 2 if dtype == torch.bool else 100, shape, generator=gen)
    return x.to(dtype).to(device)


def chosen(x, parents):
    return x[torch.arange(x.shape[0], device=x.device)[:, None], parents.long()]


def some_parents(searches, beams, n, device, seed=1, dtype=torch.int64):
    gen = torch.Generator().manual_seed(seed)
    return torch.randint(0, beams, (searches, n), generator=gen).to(dtype).to(device)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,n", [((1, 1), 1), ((2, 3), 3), ((2, 4, 1), 4), ((3, 2, 7), 5), ((2, 5, 3, 11), 5), ((2, 8, 255), 8),
                                     ((1, 4, 3, 100, 5), 4), ((2, 16, 33), 16), ((1, 31, 70), 31), ((2, 64, 19), 64), ((1, 3, 40), 200),
                                     ((2, 100, 9), 100), ((3, 1, 5000), 1)])
def test_out_of_place_and_in_place(cuda_device, dtype, shape, n):
    x = state(shape, dtype, cuda_device)
    parents = some_parents(shape[0], shape[1], n, cuda_device)
    want = chosen(x, parents)
    assert torch.equal(reorder_states(x, parents), want)
    out = torch.empty_like(want)
    assert reorder_states(x, parents.int(), out=out) is out and torch.equal(out, want)
    if n == shape[1] and n <= 64:
        assert reorder_states(x, parents, out=x) is x and torch.equal(x, want)


@pytest.mark.parametrize("order", [[0, 1, 2, 3], [3, 2, 1, 0], [1, 2, 3, 0], [0, 0, 0, 0], [3, 3, 0, 0], [1, 0, 2, 2]])
def test_orders_in_place(cuda_device, order):
    parents = torch.tensor([order, order[::-1]], device=cuda_device)
    for length in (1, 5, 16, 23, 100000):
        x = state((2, 4, length), torch.int32, cuda_device)
        want = chosen(x, parents)
        reorder_states([x], parents, out=[x])
        assert torch.equal(x, want)


def test_lists_of_states(cuda_device):
    """More than a launch takes, of different types and shapes; some empty."""
    shapes = [(3, 4, 5 * i, 1 + i % 7) for i in range(37)] + [(3, 4)]
    states = [state(s, TYPES[i % len(TYPES)], cuda_device, i) for i, s in enumerate(shapes)]
    parents = some_parents(3, 4, 4, cuda_device)
    want = [chosen(x, parents) for x in states]
    got = reorder_states(tuple(states), parents)
    assert isinstance(got, list) and all(torch.equal(a, b) for a, b in zip(got, want))
    assert reorder_states(states, parents, out=states) is states
    assert all(torch.equal(a, b) for a, b in zip(states, want))
    assert reorder_states([], parents) == []


def test_views_of_caches(cuda_device):
    """Positions in use of a longer cache, keys and values side by side, layers in one tensor."""
    parents = some_parents(2, 3, 3, cuda_device)
    cache = state((2, 3, 5, 40, 9), torch.bfloat16, cuda_device)
    used = cache[:, :, :, :17]
    whole = cache.clone()
    assert torch.equal(reorder_states(used, parents), chosen(used, parents))
    want = chosen(used, parents)
    reorder_states(used, parents, out=used)
    whole[:, :, :, :17] = want
    assert torch.equal(cache, whole)  # and what lies behind stays
    pair = state((2, 3, 20, 2, 6), torch.int32, cuda_device)
    keys, values = pair[:, :, :, 0], pair[:, :, :, 1]
    want = chosen(pair, parents)
    reorder_states([keys, values], parents, out=[keys, values])
    assert torch.equal(pair, want)
    layers = state((4, 2, 3, 50), torch.uint8, cuda_device)
    want = [chosen(x, parents) for x in layers]
    reorder_states(list(layers), parents, out=list(layers))
    assert all(torch.equal(a, b) for a, b in zip(layers, want))
    # beams that are not in the order of memory, dimensions that are not
    turned = state((3, 2, 8, 6), torch.float32, cuda_device)
    for x in (turned.transpose(0, 1), turned.transpose(0, 1).transpose(2, 3), turned.transpose(0, 1)[..., ::2],
              turned[:1, :1].expand(2, 3, 8, 6)):
        assert torch.equal(reorder_states(x, parents), chosen(x, parents))
        out = torch.empty(2, 3, *x.shape[2:], device=cuda_device)
        assert torch.equal(reorder_states(x, parents, out=out), chosen(x, parents))
    into = torch.zeros(2, 3, 5, 40, 9, dtype=torch.bfloat16, device=cuda_device)
    flat = state((2, 3, 5, 17, 9), torch.bfloat16, cuda_device)
    reorder_states(flat, parents, out=into[:, :, :, :17])
    assert torch.equal(into[:, :, :, :17], chosen(flat, parents)) and not bool(into[:, :, :, 17:].any())


def test_odd_addresses(cuda_device):
    base = state((4000,), torch.uint8, cuda_device)
    for at in (1, 2, 3, 7):
        for length in (1, 2, 15, 17, 31, 64, 99):
            x = base[at:at + 12 * length].view(3, 4, length)
            parents = some_parents(3, 4, 4, cuda_device, at)
            want, kept = chosen(x, parents), base.clone()
            reorder_states(x, parents, out=x)
            kept[at:at + 12 * length] = want.flatten()
            assert torch.equal(base, kept)


def test_parents_outside_are_zeros(cuda_device):
    x = state((2, 3, 50), torch.int64, cuda_device) + 1
    for parents in (torch.tensor([[0, -1, 2], [3, 1, 1 << 40]]), torch.tensor([[0, -1, 2], [3, 1, 1 << 30]], dtype=torch.int32)):
        parents = parents.to(cuda_device)
        there = (parents >= 0) & (parents < 3)
        want = torch.where(there[:, :, None], chosen(x, parents.clamp(0, 2)), 0)
        assert torch.equal(reorder_states(x, parents), want)
        y = x.clone()
        reorder_states(y, parents, out=y)
        assert torch.equal(y, want)


def test_no_beams_and_no_positions(cuda_device):
    x = torch.ones(2, 0, 5, device=cuda_device)
    assert torch.equal(reorder_states(x, torch.zeros(2, 3, dtype=torch.int64, device=cuda_device)), torch.zeros(2, 3, 5, device=cuda_device))
    none = torch.zeros(2, 0, dtype=torch.int64, device=cuda_device)
    assert reorder_states(x, none).shape == (2, 0, 5) and reorder_states(x, none, out=x) is x
    assert reorder_states(torch.ones(2, 4, 5, device=cuda_device), none).shape == (2, 0, 5)
    assert reorder_states(torch.ones(2, 4, 0, device=cuda_device), none + 1).shape == (2, 0, 0)
    assert reorder_states(torch.ones(0, 4, 3, device=cuda_device), torch.zeros(0, 4, dtype=torch.int32, device=cuda_device)).shape == (0, 4, 3)


def test_offsets_past_32_bits(cuda_device):
    x = torch.zeros(2, 3, (1 << 30) + 77, dtype=torch.uint8, device=cuda_device)
    x[0, 1, -1], x[1, 0, -3], x[1, 2, 5] = 11, 12, 13
    parents = torch.tensor([[1, 1, 0], [2, 0, 0]], device=cuda_device)
    y = reorder_states(x, parents)
    reorder_states(x, parents, out=x)
    for z in (x, y):
        assert z[0, :, -1].tolist() == [11, 11, 0] and z[1, :, -3].tolist() == [0, 12, 12] and z[1, :, 5].tolist() == [13, 0, 0]
        assert int(torch.count_nonzero(z)) == 5


def test_conjugates_and_negatives(cuda_device):
    x = torch.complex(torch.randn(2, 3, 4, device=cuda_device), torch.randn(2, 3, 4, device=cuda_device))
    parents = some_parents(2, 3, 3, cuda_device)
    for y in (x.conj(), x.conj().imag):
        assert torch.equal(reorder_states(y, parents).resolve_conj(), chosen(y.clone(), parents))


def test_captured(cuda_device):
    states = [state((2, 4, 100, i + 1), torch.float32, cuda_device, i) for i in range(20)]
    parents = some_parents(2, 4, 4, cuda_device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        reorder_states(states, parents, out=states)
    for turn in range(3):
        want = [chosen(x, parents) for x in states]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(states, want))
        parents.copy_(some_parents(2, 4, 4, cuda_device, turn + 5))


def test_versions_and_inference(cuda_device):
    x = state((2, 3, 4), torch.float32, cuda_device)
    parents = some_parents(2, 3, 3, cuda_device)
    version = x._version
    reorder_states(x, parents, out=x)
    assert x._version == version + 1
    with torch.inference_mode():
        y = state((2, 3, 4), torch.float32, cuda_device)
        want = chosen(y, parents)
        assert torch.equal(reorder_states(y, parents, out=y), want)


def _overlapping(t):
    base = t["x"].new_zeros(2, 3, 16)
    return base[..., :10], base[..., 6:]


REFUSED = [
    (lambda t: reorder_states(t["x"].cpu(), t["p"]), RuntimeError, "must be on CUDA"),
    (lambda t: reorder_states(t["x"], t["p"].cpu()), RuntimeError, "must be on CUDA"),
    (lambda t: reorder_states(t["x"], t["p"].float()), RuntimeError, "int32 or int64"),
    (lambda t: reorder_states(t["x"], t["p"][0]), ValueError, r"parents must be \[B, n\]"),
    (lambda t: reorder_states(5, t["p"]), RuntimeError, "list or tuple"),
    (lambda t: reorder_states([t["x"], 5], t["p"]), RuntimeError, "must be a torch.Tensor"),
    (lambda t: reorder_states(t["x"][0], t["p"]), ValueError, "states must be"),
    (lambda t: reorder_states(t["x"][0, 0], t["p"]), ValueError, "states must be"),
    (lambda t: reorder_states([t["x"], t["x"][:, :2]], t["p"]), ValueError, "of one K"),
    (lambda t: reorder_states(t["x"], t["p"], out=[t["x"]]), ValueError, "as many tensors"),
    (lambda t: reorder_states([t["x"]], t["p"], out=[]), ValueError, "as many tensors"),
    (lambda t: reorder_states([t["x"]], t["p"], out=[None]), RuntimeError, "must be a torch.Tensor"),
    (lambda t: reorder_states(t["x"], t["p"], out=t["y"].double()), ValueError, "out must be"),
    (lambda t: reorder_states(t["x"], t["p"], out=t["y"][..., :3]), ValueError, "out must be"),
    (lambda t: reorder_states(t["x"], t["p"], out=t["y"].cpu()), RuntimeError, "must be on"),
    (lambda t: reorder_states(t["x"], t["p"], out=t["y"][..., :1].expand(2, 3, 10)), ValueError, "runs that|must not overlap"),
    (lambda t: reorder_states(t["x"], t["p"], out=t["y"][:, :1].expand(2, 3, 10)), ValueError, "must not overlap"),
    (lambda t: reorder_states(t["x"], t["p"], out=t["y"].clone().requires_grad_()), ValueError, "require a gradient"),
    (lambda t: reorder_states([t["x"], t["x"]], t["p"], out=[t["x"], t["x"]]), ValueError, "share no memory"),
    (lambda t: reorder_states([t["x"], t["x"]], t["p"], out=[t["y"], t["y"]]), ValueError, "share no memory"),
    (lambda t: reorder_states(*(lambda a, b: (a, t["p"], b))(*_overlapping(t))), ValueError, "share no memory"),
    (lambda t: reorder_states(t["x"], t["p"][:, :2], out=t["x"][:, :2]), ValueError, "in place, parents|share no memory"),
    (lambda t: reorder_states(t["wide"], t["pw"], out=t["wide"]), ValueError, "at most 64 beams"),
    (lambda t: reorder_states(t["deep"], t["p"], out=t["deep"]), ValueError, "at most one dimension of runs"),
    (lambda t: reorder_states(t["p"], t["p"], out=t["p"]), ValueError, "overlap parents"),
    (lambda t: reorder_states(t["x"], torch.zeros(2, 4097, dtype=torch.int64, device="cuda")), ValueError, "at most 4096"),
]


@pytest.mark.parametrize("case", range(len(REFUSED)))
def test_refusals(cuda_device, case):
    call, kind, message = REFUSED[case]
    t = dict(x=torch.zeros(2, 3, 10, device=cuda_device), y=torch.zeros(2, 3, 10, device=cuda_device),
             p=torch.zeros(2, 3, dtype=torch.int64, device=cuda_device), wide=torch.zeros(2, 65, 4, device=cuda_device),
             pw=torch.zeros(2, 65, dtype=torch.int64, device=cuda_device),
             deep=torch.zeros(2, 3, 4, 5, 6, device=cuda_device)[:, :, :3, :4, :5])
    with pytest.raises(kind, match=message):
        call(t)
