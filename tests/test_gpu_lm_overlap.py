"""Results of process_logits that share memory with its inputs: in place, between other rows, or refused."""
import pytest
import torch

from spiky_amd import process_logits

pytestmark = pytest.mark.gpu

V = 5000


def inputs(device):
    gen = torch.Generator(device).manual_seed(1)
    return torch.randn(6, V, generator=gen, device=device)


def test_results_over_other_elements_of_an_input_are_refused(cuda_device):
    """Every check is the host's, before a launch."""
    x = inputs(cuda_device)
    flat, wide = torch.zeros(8 * V, device=cuda_device), torch.zeros(6, 2 * V, device=cuda_device)
    shifted = flat[16:16 + 6 * V].view(6, V)
    half = flat.view(torch.bfloat16)[:6 * V].view(6, V)
    mask = flat.view(torch.bool)[4 * V:4 * V + 6 * V].view(6, V)
    ids = flat.view(torch.int64)[:18].view(6, 3)
    tokens = flat.view(torch.int32)[5 * V:5 * V + 24].view(6, 4)
    out = flat[:6 * V].view(6, V)
    cases = [dict(logits=shifted), dict(logits=half), dict(logits=flat[V:7 * V].view(6, V)), dict(bias=shifted),
             dict(bias=flat[:V]), dict(mask=mask), dict(tokens=tokens, repetition_penalty=1.5),
             dict(tokens=torch.zeros(6, 3, dtype=torch.int64, device=cuda_device), lengths=flat.view(torch.int32)[:6]),
             dict(tokens=torch.zeros(6, 3, dtype=torch.int64, device=cuda_device), prompt_lengths=flat.view(torch.int32)[-2 * V - 6:-2 * V]),
             dict(bias_ids=ids, bias_values=torch.zeros(6, 3, device=cuda_device)),
             dict(bias_ids=torch.zeros(6, 3, dtype=torch.int64, device=cuda_device), bias_values=flat[9:27].view(6, 3)),
             *(dict([(n, flat[V:V + 6])]) for n in ("temperature", "repetition_penalty", "presence_penalty", "frequency_penalty"))]
    for case in cases:
        with pytest.raises(ValueError, match="overlap|another view"):
            process_logits(**{**dict(logits=x, out=out), **case})
    with pytest.raises(ValueError, match="overlap"):
        process_logits(wide[:, :V], out=wide[:, 8:V + 8])


def test_results_beside_the_logits(cuda_device):
    """In place, in the rows between, in the other half of them, in one row, over a bias of their shape."""
    x = inputs(cuda_device)
    bias = torch.randn(6, V, device=cuda_device)
    want = process_logits(x, bias=bias, temperature=0.5)
    for rows in (slice(None), slice(0, 1)):
        wide = torch.zeros(6, 3, V, device=cuda_device)
        wide[:, 1] = x
        given = wide[rows, 1]
        assert torch.equal(process_logits(given, bias=bias[rows], temperature=0.5, out=wide[rows, 2]), want[rows])
        assert torch.equal(wide[:, 1], x)
        process_logits(given, bias=bias[rows], temperature=0.5, out=wide[rows, 1])
        assert torch.equal(given, want[rows])
    row = torch.zeros(2, V, device=cuda_device)
    row[0] = x[0]
    process_logits(row[:1], bias=bias[:1], temperature=0.5, out=row.as_strided((1, V), (7 * V, 1)))
    assert torch.equal(row[:1], want[:1])
    over = bias.clone()
    assert torch.equal(process_logits(x, bias=over, temperature=0.5, out=over), want)
