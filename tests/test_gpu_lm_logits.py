"""Processed logits on the GPU against their definition in 64 bits."""
import math

import pytest
import torch

from spiky_amd import process_logits
import lm_plain

pytestmark = pytest.mark.gpu

# bias, sparse biases, penalty factor and its reciprocal, two products and a difference of penalties,
# the temperature's reciprocal and product: a dozen roundings
STEPS = 16

TYPES = [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
         (torch.bfloat16, torch.float32), (torch.float16, torch.float32)]


def pack(mask):
    """Truth values [..., V] as int32 words, lowest bit first."""
    V = mask.shape[-1]
    m = torch.nn.functional.pad(mask.to(torch.int64), (0, -V % 32)).reshape(*mask.shape[:-1], -1, 32)
    w = (m << torch.arange(32, device=mask.device)).sum(-1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)


def make(B, V, L=0, K=0, token=torch.int64, seed=0):
    gen = torch.Generator().manual_seed(seed)
    s = {"x": torch.randn(B, V, generator=gen) * 4}
    if L:
        s["tokens"] = (torch.rand(B, L, generator=gen) ** 3 * V).to(token)
        s["lengths"] = torch.randint(0, L + 1, (B,), generator=gen)
        s["prompts"] = (s["lengths"] * torch.rand(B, generator=gen)).to(torch.int64)
    if K:
        s["ids"] = (torch.rand(B, K, generator=gen) ** 2 * V).to(token)
        s["values"] = torch.randn(B, K, generator=gen) * 3
    s["gen"] = gen
    return s


def check(dev, x, out=None, dtype=None, mask=None, packed=False, **kw):
    names = dict(tokens="tokens", lengths="lengths", prompts="prompt_lengths", rho="repetition_penalty",
                 presence="presence_penalty", frequency="frequency_penalty", bias="bias", ids="bias_ids",
                 values="bias_values", temperature="temperature")
    want, size = lm_plain.logits(x, mask=mask, **kw)
    given = {names[k]: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in kw.items()}
    if mask is not None:
        given["mask"] = (pack(mask) if packed else mask).to(dev)
    x = x if x.device == dev else x.to(dev)
    got = process_logits(x, out=out, dtype=dtype, **given)
    assert got.dtype == (dtype or (x.dtype if out is None else out.dtype))
    lm_plain.near(got, want, size, STEPS)
    return got


@pytest.mark.parametrize("dtype,out", TYPES)
@pytest.mark.parametrize("V", [1, 7, 8, 31, 33, 256, 2047, 2049, 8193, 50001])
def test_vocabularies(cuda_device, dtype, out, V):
    s = make(3, V, L=200, K=20)
    check(cuda_device, s["x"].to(dtype), dtype=out, tokens=s["tokens"], lengths=s["lengths"], prompts=s["prompts"],
          rho=1.3, presence=0.5, frequency=0.25, ids=s["ids"], values=s["values"], temperature=0.8,
          bias=torch.randn(V), mask=torch.rand(3, V, generator=s["gen"]) < 0.5, packed=True)


@pytest.mark.parametrize("token", [torch.int32, torch.int64])
@pytest.mark.parametrize("B,V,L", [(1, 100, 1), (2, 64, 5000), (70, 300, 17), (1, 20000, 40000), (5, 130000, 300)])
def test_histories(cuda_device, token, B, V, L):
    s = make(B, V, L, token=token)
    rows = {k: torch.rand(B, generator=s["gen"]) for k in ("presence", "frequency")}
    check(cuda_device, s["x"], tokens=s["tokens"], lengths=s["lengths"].to(token), prompts=s["prompts"].to(torch.int32),
          rho=1.0 + torch.rand(B, generator=s["gen"]), temperature=torch.rand(B, generator=s["gen"]) + 0.5, **rows)
    check(cuda_device, s["x"], tokens=s["tokens"], rho=0.7, presence=-0.5, frequency=-0.1)
    check(cuda_device, s["x"], tokens=s["tokens"], prompts=s["prompts"], rho=1.5, presence=1.0)


def test_lengths_and_tokens_out_of_range(cuda_device):
    s = make(6, 500, 40)
    tokens = s["tokens"]
    tokens[:, ::3] = torch.tensor([-1, 500, 1 << 40, -(1 << 40), (1 << 32) + 3, -500])[:, None]
    lengths = torch.tensor([0, 1, 40, 41, -3, 1 << 40])
    prompts = torch.tensor([5, 0, -7, 50, 2, 20])
    check(cuda_device, s["x"], tokens=tokens, lengths=lengths, prompts=prompts, rho=2.0, presence=0.25, frequency=0.5)
    check(cuda_device, s["x"], tokens=tokens[:, :0], rho=2.0, presence=0.25)


@pytest.mark.parametrize("K", [1, 63, 64, 65, 300, 1000])
@pytest.mark.parametrize("V", [5, 3000, 40000])
def test_sparse_biases_add_up(cuda_device, K, V):
    s = make(2, V, K=K)
    s["ids"][1, : K // 2] = 3
    s["ids"][0, -1] = -1
    check(cuda_device, s["x"], ids=s["ids"], values=s["values"])
    check(cuda_device, s["x"], ids=s["ids"][1].to(torch.int32), values=s["values"][0], bias=torch.randn(2, V).to(torch.bfloat16))


@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("V", [1, 30, 32, 100, 9001])
def test_masks(cuda_device, packed, V):
    x = make(4, V)["x"]
    x[0], x[1, 0] = float("nan"), float("inf")
    mask = torch.rand(4, V) < 0.5
    mask[0], mask[2], mask[3] = False, False, True
    got = check(cuda_device, x, mask=mask, packed=packed, temperature=0.5)
    assert (got[0] == -math.inf).all() and (got[2] == -math.inf).all()
    check(cuda_device, x, mask=mask[1], packed=packed)


def test_values_at_the_ends(cuda_device):
    """-inf stays, the lowest value divided by a temperature becomes -inf, NaN stays NaN."""
    low = torch.finfo(torch.float32).min
    x = torch.tensor([[-math.inf, low, math.inf, math.nan, 0.0, -0.0, 1.0, -1.0]] * 2)
    tokens = torch.arange(8).repeat(2, 1)
    got = process_logits(x.to(cuda_device), tokens=tokens.to(cuda_device), repetition_penalty=2.0, temperature=0.5,
                         presence_penalty=0.25).cpu()
    want = [-math.inf, -math.inf, math.inf, math.nan, -0.5, -0.5, 0.5, -4.5]
    assert torch.equal(got[0].nan_to_num(7.0, math.inf, -math.inf), torch.tensor(want).nan_to_num(7.0, math.inf, -math.inf))


def test_temperature_zero_leaves_a_row(cuda_device):
    x = make(3, 100)["x"]
    check(cuda_device, x, temperature=torch.tensor([0.0, 0.5, -1.0]))
    check(cuda_device, x, temperature=0.0)


def test_strided_rows_and_in_place(cuda_device):
    s = make(5, 1001, 50, 9)
    wide = torch.randn(5, 4, 1001, device=cuda_device)
    kw = dict(tokens=s["tokens"], rho=1.2, frequency=0.3, ids=s["ids"], values=s["values"], temperature=2.0)
    check(cuda_device, wide[:, -1], **kw)
    check(cuda_device, wide[:, 1, 3:900], tokens=s["tokens"], rho=1.2)
    check(cuda_device, torch.randn(900, 5, device=cuda_device).t(), tokens=s["tokens"], rho=1.2)
    tokens = torch.randint(0, 1001, (5, 3, 60))
    check(cuda_device, wide[:, 0], tokens=tokens[:, 1], rho=1.2, lengths=torch.tensor([0, 1, 30, 59, 60]))
    check(cuda_device, wide[:, 0], tokens=tokens.transpose(1, 2)[:, :, 0], rho=1.2)
    x = wide[:, 2]
    before = wide.clone()
    want, size = lm_plain.logits(x, **kw)
    given = {k: v.to(cuda_device) if isinstance(v, torch.Tensor) else v for k, v in kw.items()}
    got = process_logits(x, out=x, tokens=given["tokens"], repetition_penalty=1.2, frequency_penalty=0.3,
                         bias_ids=given["ids"], bias_values=given["values"], temperature=2.0)
    assert got is x
    lm_plain.near(x, want, size, STEPS)
    assert torch.equal(wide[:, [0, 1, 3]], before[:, [0, 1, 3]])


def test_many_rows(cuda_device):
    s = make(70000, 40, 3)
    check(cuda_device, s["x"][:200], tokens=s["tokens"][:200], rho=1.5)
    got = process_logits(s["x"].to(cuda_device), tokens=s["tokens"].to(cuda_device), repetition_penalty=1.5)
    tail, size = lm_plain.logits(s["x"][-5000:], tokens=s["tokens"][-5000:], rho=1.5)
    lm_plain.near(got[-5000:], tail, size, STEPS)


def test_a_large_batch_passes_32_bits(cuda_device):
    B, V = 16500, 262144  # 2^32 entries and some, of two bytes
    x = torch.zeros(B, V, dtype=torch.bfloat16, device=cuda_device)
    x[-1] = torch.arange(V, device=cuda_device) % 128
    got = process_logits(x, out=x, temperature=0.5, tokens=torch.full((B, 1), V - 1, device=cuda_device), presence_penalty=1.0)
    assert torch.equal(got[-1, :-1].float(), 2.0 * (torch.arange(V - 1, device=cuda_device) % 128))
    assert float(got[-1, -1]) == 252.0 and float(got[-2, -1]) == -2.0


def test_results_do_not_vary_and_replay(cuda_device):
    s = {k: v.to(cuda_device) if isinstance(v, torch.Tensor) else v for k, v in make(4, 5000, 3000, 200).items()}

    def call():
        return process_logits(s["x"], tokens=s["tokens"], lengths=s["lengths"], prompt_lengths=s["prompts"],
                              repetition_penalty=1.1, presence_penalty=0.2, frequency_penalty=0.1, bias_ids=s["ids"],
                              bias_values=s["values"], temperature=0.9)

    first = call()
    assert torch.equal(first, call())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = call()
    for k in range(3):
        s["x"].normal_()
        s["tokens"].random_(0, 5000)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, call())


def test_empty(cuda_device):
    assert process_logits(torch.zeros(0, 9, device=cuda_device)).shape == (0, 9)
    assert process_logits(torch.zeros(3, 0, device=cuda_device)).shape == (3, 0)
