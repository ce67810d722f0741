"""What the language-model operators refuse of device tensors; every check is the host's, before a launch."""
import pytest
import torch

from spiky_amd import counter_dropout, process_logits, residual_norm

pytestmark = pytest.mark.gpu


def tensors(device):
    x = torch.zeros(4, 6, 8, device=device)
    return dict(x=x, h=x.to(torch.bfloat16), half=x.to(torch.float16), d=x.double(), w=torch.ones(8, device=device),
                i=torch.zeros(4, 8, dtype=torch.int64, device=device), cpu=torch.zeros(4, 6, 8), l=x[:, 0],
                wh=torch.ones(8, device=device, dtype=torch.bfloat16))


DROPOUT = [
    (lambda t: counter_dropout(t["d"], 0.5, 1), RuntimeError, "must be float32, bfloat16 or float16"),
    (lambda t: counter_dropout(t["x"], 1.5, 1), ValueError, "between 0 and 1"),
    (lambda t: counter_dropout(t["x"], float("nan"), 1), ValueError, "between 0 and 1"),
    (lambda t: counter_dropout(t["x"], 0.5, t["i"]), RuntimeError, r"\[seed, offset\]"),
    (lambda t: counter_dropout(t["x"], 0.5, torch.zeros(2, dtype=torch.int64)), RuntimeError, "must be on CUDA"),
    (lambda t: counter_dropout(t["x"], 0.5, t["i"][0, :2], 3), ValueError, "second element of a seed tensor"),
    (lambda t: counter_dropout(t["x"], 0.5, 1.5), TypeError, "integer"),
    (lambda t: counter_dropout(t["x"], "half", 1), TypeError, "real number"),
]
RESIDUAL = [
    (lambda t: residual_norm(t["x"]), ValueError, "neither a branch nor a pre_norm"),
    (lambda t: residual_norm(t["x"][0, 0, 0], pre_norm="rms"), ValueError, "at least one dimension"),
    (lambda t: residual_norm(t["x"], gate=t["w"], pre_norm="rms"), ValueError, "needs a branch"),
    (lambda t: residual_norm(t["x"], t["x"], pre_norm="batch"), ValueError, "'rms' or 'layer'"),
    (lambda t: residual_norm(t["x"], t["x"], pre_weight=t["w"]), ValueError, "need a pre_norm"),
    (lambda t: residual_norm(t["x"], t["x"][:, 1:]), ValueError, "for a residual of"),
    (lambda t: residual_norm(t["h"], t["x"]), RuntimeError, "does not go with"),
    (lambda t: residual_norm(t["h"], t["half"]), RuntimeError, "does not go with"),
    (lambda t: residual_norm(t["x"], t["h"], dtype=torch.float16), ValueError, "dtype is the branch's"),
    (lambda t: residual_norm(t["x"], t["cpu"]), RuntimeError, "must be on CUDA"),
    (lambda t: residual_norm(t["x"], t["x"], pre_norm="rms", pre_weight=t["w"][:7]), ValueError, "must have shape"),
    (lambda t: residual_norm(t["x"], t["x"], pre_norm="rms", pre_weight=t["wh"]), RuntimeError, "must be float32 or"),
    (lambda t: residual_norm(t["x"], t["h"], post_norm="rms", post_weight=t["wh"], pre_norm="rms", pre_weight=t["w"]),
     RuntimeError, "one type"),
    (lambda t: residual_norm(t["x"], t["x"], gate=t["w"][:3]), ValueError, "does not broadcast"),
    (lambda t: residual_norm(t["x"], t["x"], gate=t["wh"]), RuntimeError, "gate must be float32"),
    (lambda t: residual_norm(t["x"], t["x"], dropout_p=-0.5), ValueError, "between 0 and 1"),
    (lambda t: residual_norm(t["x"], t["x"], post_norm="rms", post_eps="small"), TypeError, "real number"),
]
LOGITS = [
    (lambda t: process_logits(t["x"]), ValueError, r"must be \[B, V\]"),
    (lambda t: process_logits(t["l"], dtype=torch.float16), ValueError, "dtype must be"),
    (lambda t: process_logits(t["l"], out=t["l"][:2]), ValueError, "out must be"),
    (lambda t: process_logits(t["l"].clone(), out=torch.zeros(8, 4, device="cuda").t()), ValueError, "contiguous columns"),
    (lambda t: process_logits(t["l"], tokens=t["i"][0]), ValueError, r"tokens must be"),
    (lambda t: process_logits(t["l"], tokens=t["i"][:3]), ValueError, "tokens must be"),
    (lambda t: process_logits(t["l"], tokens=t["l"]), RuntimeError, "int32 or int64"),
    (lambda t: process_logits(t["l"], lengths=t["i"][:, 0]), ValueError, "lengths need tokens"),
    (lambda t: process_logits(t["l"], tokens=t["i"], lengths=t["i"][0, :3]), ValueError, "lengths must have shape"),
    (lambda t: process_logits(t["l"], repetition_penalty=0.0), ValueError, "must be positive"),
    (lambda t: process_logits(t["l"], temperature=t["w"]), ValueError, "must be a number or have shape"),
    (lambda t: process_logits(t["l"], temperature=t["i"][:, 0]), RuntimeError, "floating point"),
    (lambda t: process_logits(t["l"], bias=t["w"][:7]), ValueError, "bias must be"),
    (lambda t: process_logits(t["l"], bias_ids=t["i"]), ValueError, "go together"),
    (lambda t: process_logits(t["l"], bias_ids=t["i"], bias_values=t["l"][:, :7]), ValueError, "shape of bias_ids"),
    (lambda t: process_logits(t["l"], bias_ids=t["i"], bias_values=t["l"].half()), RuntimeError, "must be float32"),
    (lambda t: process_logits(t["l"], mask=t["l"]), RuntimeError, "bool or int32"),
    (lambda t: process_logits(t["l"], mask=t["l"][:, :7] > 0), ValueError, "mask must be"),
    (lambda t: process_logits(t["l"], mask=t["i"].int()), ValueError, "mask must be"),
]


@pytest.mark.parametrize("call,error,message", DROPOUT + RESIDUAL + LOGITS)
def test_refused(cuda_device, call, error, message):
    with pytest.raises(error, match=message):
        call(tensors(cuda_device))
