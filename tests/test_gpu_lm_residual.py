"""The residual join on the GPU against its formulas in 64 bits, and against differences."""
import pytest
import torch

from spiky_amd import ResidualNorm, counter_dropout, residual_norm
import lm_plain

pytestmark = pytest.mark.gpu

# Half steps of float32 that a value may be off, relative to the magnitude lm_plain.join keeps for
# it.  A row's sum runs over at most 32 values in a lane, 6 exchanges and 16 waves; a sum of squares
# of positive terms is off by as many half steps, its root by half of them.  A chain of forward and
# backward has four such sums and about 30 single operations.
FORWARD = 2 * (32 + 6 + 16) + 20
BACKWARD = 4 * (32 + 6 + 16) + 40


def tensors(rows, D, act, res, par, post, pre, gate, biases, gate_rows=1, branch=True, seed=1):
    gen = torch.Generator().manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen)

    t = {"r": (normal(rows, D) * 2).to(res), "a": normal(rows, D).to(act) if branch else None}
    for norm, w, b in ((post, "w1", "b1"), (pre, "w2", "b2")):
        t[w] = (normal(D) * 0.3 + 1).to(par) if norm else None
        t[b] = normal(D).to(par) if norm and biases else None
    t["g"] = None
    if gate == "channel":
        t["g"] = normal(D).to(par)
    elif gate == "rows":
        t["g"] = normal(rows // gate_rows, D).to(act)
    elif gate == "full":
        t["g"] = normal(rows, D).to(act)
    t["d_out"], t["d_normed"] = normal(rows, D).to(res), normal(rows, D).to(act) if pre else None
    return t


def shared(gate, rows, D):
    """A gate's rows repeated for every row it stands for."""
    if gate is None:
        return None
    g = gate.reshape(-1, D)
    return g.repeat_interleave(rows // g.shape[0], 0)


def check(device, rows, D, act=torch.float32, res=None, par=torch.float32, post="rms", pre="rms", gate=None,
          biases=False, gate_rows=1, branch=True, train=True, leave=(), **how):
    res = act if res is None else res
    t = tensors(rows, D, act, res, par, post, pre, gate, biases, gate_rows, branch)
    how = dict(how, post_norm=post, pre_norm=pre)
    names = {"r": None, "a": None, "w1": "post_weight", "b1": "post_bias", "g": "gate", "w2": "pre_weight", "b2": "pre_bias"}
    shape = (rows // gate_rows, gate_rows, D)
    d = {k: None if v is None else v.to(device) for k, v in t.items()}
    for k in ("r", "a", "d_out", "d_normed"):
        d[k] = None if d[k] is None else d[k].reshape(shape)
    if gate == "rows":
        d["g"] = d["g"].reshape(shape[0], 1, D)
    elif gate == "full":
        d["g"] = d["g"].reshape(shape)
    if train:
        for k in names:
            if d[k] is not None:
                d[k].requires_grad_()
    z, h = residual_norm(d["r"], d["a"], **{n: d[k] for k, n in names.items() if n}, **how)
    plain = {k: t[k] for k in names}
    plain["g"] = shared(t["g"], rows, D)
    d_out = None if "out" in leave or not branch else t["d_out"]
    d_normed = None if "normed" in leave else t["d_normed"]
    want, size = lm_plain.join(plain, how, *((d_out, d_normed) if train else (None, None)))
    if branch:
        assert z.dtype == res
        lm_plain.near(z, want["z"], size["z"], FORWARD, "out")
    else:
        assert z is d["r"]
    if pre:
        assert h.dtype == act
        lm_plain.near(h, want["h"], size["h"], FORWARD, "normed")
    else:
        assert h is None
    if not train:
        return
    outs = [(z, d["d_out"])] if d_out is not None else []
    outs += [(h, d["d_normed"])] if d_normed is not None else []
    wanted = [k for k in names if d[k] is not None]
    got = dict(zip(wanted, torch.autograd.grad([o for o, _ in outs], [d[k] for k in wanted], [g for _, g in outs])))
    for k in wanted:
        assert got[k].dtype == d[k].dtype and got[k].shape == d[k].shape
        w, s = want.get(k), size.get(k)
        if w is None:  # a pre norm's parameters without a gradient of its output
            assert not got[k].any()
            continue
        steps = BACKWARD
        if k == "g" and gate != "full":
            w, s = w.reshape(d[k].reshape(-1, D).shape[0], -1, D).sum(1), s.reshape(d[k].reshape(-1, D).shape[0], -1, D).sum(1)
        if k not in ("r", "a"):
            steps += rows  # a sum over the rows in any order is off by fewer half steps than it has terms
        lm_plain.near(got[k].reshape(w.shape), w, s, steps, "gradient of " + k)


TYPES = [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
         (torch.bfloat16, torch.float32), (torch.float16, torch.float32)]


@pytest.mark.parametrize("act,res", TYPES)
@pytest.mark.parametrize("D", [1, 3, 8, 16, 63, 130, 257, 512, 1000, 1025, 2048, 4100, 8200])
def test_widths(cuda_device, act, res, D):
    check(cuda_device, 6, D, act, res, dropout_p=0.2, seed=3, offset=4)


@pytest.mark.parametrize("D", [16385, 40000])
@pytest.mark.parametrize("act,res", [TYPES[0], TYPES[3]])
def test_wide_rows(cuda_device, act, res, D):
    check(cuda_device, 3, D, act, res, post="layer", pre="layer", gate="channel", biases=True, dropout_p=0.2, seed=3)


@pytest.mark.parametrize("post", [None, "rms", "layer"])
@pytest.mark.parametrize("pre", [None, "rms", "layer"])
@pytest.mark.parametrize("gate", [None, "channel", "rows", "full"])
@pytest.mark.parametrize("train", [True, False])
def test_parts(cuda_device, post, pre, gate, train):
    check(cuda_device, 24, 200, post=post, pre=pre, gate=gate, biases=True, gate_rows=4, train=train,
          residual_scale=0.75, branch_scale=-1.5)


@pytest.mark.parametrize("par", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,gate_rows", [(1, 1), (2, 1), (5, 5), (40, 40), (96, 3), (1000, 10), (1200, 600), (2051, 1),
                                            (5000, 5000), (6000, 2)])
def test_rows_of_a_gate(cuda_device, par, rows, gate_rows):
    check(cuda_device, rows, 72, torch.bfloat16, torch.float32, par, gate="rows", gate_rows=gate_rows, dropout_p=0.1,
          seed=8, biases=True)


@pytest.mark.parametrize("rows", [1, 3, 5000, 20000])
def test_column_sums_over_many_rows(cuda_device, rows):
    check(cuda_device, rows, 40, post="layer", pre="layer", gate="channel", biases=True)


@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("act,res", [TYPES[0], TYPES[1]])
@pytest.mark.parametrize("D", [200, 20000])
def test_norm_alone(cuda_device, norm, act, res, D):
    check(cuda_device, 9, D, act, res, post=None, pre=norm, branch=False, biases=True)


@pytest.mark.parametrize("leave", ["out", "normed"])
@pytest.mark.parametrize("D", [100, 17000])
def test_one_output_without_a_gradient(cuda_device, leave, D):
    check(cuda_device, 10, D, post="layer", pre="layer", gate="channel", biases=True, leave=(leave,))


def test_parameters_may_be_absent(cuda_device):
    a, r = torch.randn(4, 300, device=cuda_device), torch.randn(4, 300, device=cuda_device)
    z, h = residual_norm(r, a, post_norm="rms", pre_norm="layer")
    want, size = lm_plain.join(dict(r=r, a=a, w1=None, b1=None, g=None, w2=None, b2=None), dict(post_norm="rms", pre_norm="layer"))
    lm_plain.near(z, want["z"], size["z"], FORWARD)
    lm_plain.near(h, want["h"], size["h"], FORWARD)


def test_dropout_is_counter_dropouts(cuda_device):
    a, r = torch.randn(31, 101, device=cuda_device), torch.zeros(31, 101, device=cuda_device)
    z, _ = residual_norm(r, a, dropout_p=0.35, seed=5, offset=6)
    assert torch.equal(z, counter_dropout(a, 0.35, 5, 6))
    state = torch.tensor([5, 6], dtype=torch.int64, device=cuda_device)
    assert torch.equal(z, residual_norm(r, a, dropout_p=0.35, seed=state)[0])
    assert torch.equal(residual_norm(r + 1, a, dropout_p=1.0)[0], r + 1)


def test_dropped_infinities_leave_the_residual(cuda_device):
    a = torch.full((8, 64), float("inf"), device=cuda_device)
    r = torch.ones(8, 64, device=cuda_device, requires_grad=True)
    a.requires_grad_()
    z, _ = residual_norm(r, a, dropout_p=0.5, seed=2)
    keep = lm_plain.kept(8, 64, 0.5, 2, 0)
    assert torch.equal(z.cpu(), torch.where(keep, float("inf"), 1.0))
    (da,) = torch.autograd.grad(z, a, torch.ones_like(z))
    assert torch.equal(da.cpu(), keep.float() * 2)


def test_special_rows(cuda_device):
    """A row of zeros is divided by the root of eps; NaN and infinities stay in their row."""
    a = torch.randn(6, 96, device=cuda_device)
    a[1], a[3, 5], a[4, 7] = 0.0, float("nan"), float("inf")
    r = torch.randn(6, 96, device=cuda_device)
    z, h = residual_norm(r, a, post_norm="rms", pre_norm="rms")
    assert torch.equal(z[1], r[1])
    assert torch.isnan(z[3]).all() and torch.isnan(h[3]).all()
    clean = [0, 1, 2, 5]
    want = residual_norm(r[clean], a[clean], post_norm="rms", pre_norm="rms")
    assert torch.equal(z[clean], want[0]) and torch.equal(h[clean], want[1])


@pytest.mark.parametrize("act", [torch.float32, torch.bfloat16])
def test_strides_and_broadcast_gates(cuda_device, act):
    base = torch.randn(4, 6, 3, 56, device=cuda_device).to(act)
    views = [(base[:, 1], base[:, 2]), (base[..., 0, :], base[:, :, 1]), (base.transpose(0, 1), base.transpose(1, 0)),
             (base[..., 3:33], base[..., 5:35]), (base[..., ::2], base[..., 1::2]), (base[:1, 0], base[1, :1])]
    for r, a in views:
        D = a.shape[-1]
        gates = [None, torch.randn(D, device=cuda_device), torch.randn(a.shape[-2], 1, device=cuda_device),
                 torch.randn(a.shape[-2], D, device=cuda_device), torch.randn(a.shape[0], *[1] * (a.dim() - 2), D, device=cuda_device)]
        w = torch.randn(2, D, device=cuda_device)
        for g in gates:
            how = dict(post_norm="rms", pre_norm="layer", post_weight=w[0], pre_weight=w[1], dropout_p=0.1, seed=1)
            z, h = residual_norm(r, a, gate=g, **how)
            full = None if g is None else g.expand(a.shape).contiguous()
            z2, h2 = residual_norm(r.contiguous(), a.contiguous(), gate=full, **how)
            assert torch.equal(z, z2) and torch.equal(h, h2)


def test_gradients_of_broadcast_gates_and_strided_outputs(cuda_device):
    r, a = torch.randn(3, 5, 64, device=cuda_device), torch.randn(3, 5, 64, device=cuda_device)
    dz = torch.randn(64, 5, 3, device=cuda_device).permute(2, 1, 0)
    for shape in ((64,), (1,), (5, 64), (5, 1), (3, 1, 64), (3, 1, 1), (3, 5, 64)):
        g = torch.randn(shape, device=cuda_device, requires_grad=True)
        z, _ = residual_norm(r, a, gate=g)
        (dg,) = torch.autograd.grad(z, g, dz)
        want = (a.double() * dz.double()).sum_to_size(shape)
        size = (a.double() * dz.double()).abs().sum_to_size(shape)
        lm_plain.near(dg, want.cpu(), size.cpu(), BACKWARD + 960, str(shape))


def test_gradients_are_the_slopes(cuda_device):
    """Central differences of a weighted sum of both outputs, in 32 bits: the difference of two sums of
    about 100 terms of size 1 is off by about 100 half steps, which a step of 2^-8 makes 100 * 2^-24 * 2^8,
    beside a third derivative times 2^-16."""
    torch.manual_seed(3)
    t = {k: torch.randn(*s, device=cuda_device) for k, s in
         dict(r=(2, 24), a=(2, 24), w1=(24,), b1=(24,), g=(24,), w2=(24,), b2=(24,)).items()}
    cz, ch = torch.randn(2, 24, device=cuda_device), torch.randn(2, 24, device=cuda_device)

    def f(t):
        z, h = residual_norm(t["r"], t["a"], post_norm="layer", post_weight=t["w1"], post_bias=t["b1"], gate=t["g"],
                             pre_norm="rms", pre_weight=t["w2"], pre_bias=t["b2"], residual_scale=0.7, dropout_p=0.2, seed=4)
        return (cz.double() * z.double()).sum() + (ch.double() * h.double()).sum()

    leaves = {k: v.clone().requires_grad_() for k, v in t.items()}
    grads = dict(zip(leaves, torch.autograd.grad(f(leaves), list(leaves.values()))))
    step = 2.0 ** -8
    for k, v in t.items():
        for i in range(0, v.numel(), 5):
            up, down = v.clone(), v.clone()
            up.view(-1)[i] += step
            down.view(-1)[i] -= step
            slope = float(f({**t, k: up}) - f({**t, k: down})) / (2 * step)
            got = float(grads[k].reshape(-1)[i])
            assert abs(got - slope) < 100 * 2.0 ** -16 + 2.0 ** -16 * 64 * max(1.0, abs(got)), (k, i, got, slope)


def test_results_do_not_vary(cuda_device):
    t = tensors(3000, 136, torch.bfloat16, torch.float32, torch.float32, "layer", "rms", "channel", True)
    t = {k: None if v is None else v.to(cuda_device) for k, v in t.items()}
    runs = []
    for _ in range(3):
        leaves = {k: t[k].clone().requires_grad_() for k in ("r", "a", "w1", "b1", "g", "w2", "b2")}
        z, h = residual_norm(leaves["r"], leaves["a"], post_norm="layer", post_weight=leaves["w1"], post_bias=leaves["b1"],
                             gate=leaves["g"], pre_norm="rms", pre_weight=leaves["w2"], pre_bias=leaves["b2"])
        runs.append([z, h, *torch.autograd.grad([z, h], list(leaves.values()), [t["d_out"], t["d_normed"]])])
    for other in runs[1:]:
        assert all(torch.equal(x, y) for x, y in zip(runs[0], other))


def test_empty(cuda_device):
    r, a = (torch.zeros(0, 8, device=cuda_device, requires_grad=True) for _ in range(2))
    w = torch.ones(8, device=cuda_device, requires_grad=True)
    z, h = residual_norm(r, a, pre_norm="rms", pre_weight=w)
    grads = torch.autograd.grad([z, h], [r, a, w], [torch.zeros_like(z), torch.zeros_like(h)])
    assert z.shape == (0, 8) and not grads[2].any()


def test_captured_training_step(cuda_device):
    """Forward and backward in one graph, replayed with other inputs, against the eager step."""
    t = tensors(70, 264, torch.bfloat16, torch.float32, torch.float32, "rms", "rms", "channel", False)
    t = {k: None if v is None else v.to(cuda_device) for k, v in t.items()}
    leaves = [t[k].requires_grad_() for k in ("r", "a", "w1", "g", "w2")]
    state = torch.tensor([3, 0], dtype=torch.int64, device=cuda_device)

    def step():
        z, h = residual_norm(t["r"], t["a"], post_norm="rms", post_weight=t["w1"], gate=t["g"], dropout_p=0.3, seed=state,
                             pre_norm="rms", pre_weight=t["w2"])
        grads = torch.autograd.grad([z, h], leaves, [t["d_out"], t["d_normed"]])
        return [z.detach(), h.detach(), *grads]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for k in range(3):
        with torch.no_grad():
            state[1] = k
            t["a"].normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(captured, step()))


def test_module(cuda_device):
    m = ResidualNorm(96, post_norm="rms", pre_norm="layer", bias=True, gate=0.1, dropout_p=0.2, seed=5, device=cuda_device)
    r, a = torch.randn(2, 7, 96, device=cuda_device), torch.randn(2, 7, 96, device=cuda_device)
    z, h = m(r, a)
    how = dict(post_norm="rms", post_weight=m.post_weight, post_bias=m.post_bias, gate=m.gate, pre_norm="layer",
               pre_weight=m.pre_weight, pre_bias=m.pre_bias)
    z2, h2 = residual_norm(r, a, dropout_p=0.2, seed=5, offset=1, **how)
    assert torch.equal(z, z2) and torch.equal(h, h2)
    (z.sum() + h.square().sum()).backward()
    assert all(p.grad is not None for p in m.parameters()) and len(list(m.parameters())) == 5
    z, h = m.eval()(r, a)
    z2, h2 = residual_norm(r, a, **how)
    assert torch.equal(z, z2) and torch.equal(h, h2)
    other = ResidualNorm(96, post_norm="rms", pre_norm="layer", bias=True, gate=0.1, dropout_p=0.2)
    other.load_state_dict(m.state_dict())
    assert other.calls == 1 and other.seed == 5
