"""What the operators' modules share."""
import torch


def check_probability(p):
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout probability must be between 0 and 1, got {p}")


class CountedMasks:
    """The seed and offset of a module's masks: call number n in training has offset n.

    The number is Python's, or, after mask_counters, an element of `counter`, an int64 tensor of
    [seed, offset] that the operators read and the program advances."""

    counter = None
    counter_version = None  # of the counter in the last forward pass

    def count_masks(self, seed):
        self.seed, self.calls = int(seed), 0

    def get_extra_state(self):
        if self.counter is None:
            return {"seed": self.seed, "calls": self.calls}
        seed, offset = self.counter.tolist()
        return {"seed": seed, "calls": offset - 1}

    def set_extra_state(self, state):
        self.seed, self.calls = int(state["seed"]), int(state["calls"])
        if self.counter is not None:
            self.counter.copy_(self.next_count(state))

    def __getstate__(self):
        # copies and pickles count for themselves: nobody advances a copy of the counter
        state = dict(self.__dict__)
        state.update(self.get_extra_state())
        for name in ("counter", "counter_version"):
            state.pop(name, None)
        return state

    @staticmethod
    def next_count(state):
        """[seed, offset of the next call] from a saved state."""
        seed = (int(state["seed"]) + (1 << 63)) % (1 << 64) - (1 << 63)
        return torch.tensor([seed, int(state["calls"]) + 1], dtype=torch.int64)

    def next_mask(self, x):
        """(seed, offset) of a call in training on x."""
        recomputed = torch._C._current_graph_task_id() != -1  # inside a backward pass (torch.utils.checkpoint)
        if self.counter is not None:
            version = 0 if self.counter.is_inference() else self.counter._version
            if not recomputed:
                self.counter_version = version
            elif self.counter_version not in (None, version):
                raise RuntimeError("mask counters have changed since the forward pass that a backward pass repeats: "
                                   "advance them after the backward pass")
            return self.counter, 0
        if recomputed:
            # counted again, its mask would be another one
            raise RuntimeError("dropout inside a backward pass cannot tell which call it repeats: give the model "
                               "counters with spiky_amd.mask_counters, or pass seed and offset to the functions")
        if x.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the number of a captured dropout would be the same in every replay: give the model "
                               "counters with spiky_amd.mask_counters, or pass a seed tensor to the functions")
        self.calls += 1
        return self.seed, self.calls


def mask_counters(model, device):
    """An int64 tensor [n, 2] on `device` that holds [seed, offset] of the next masks of each CounterDropout
    and ResidualNorm of `model`, in the order of its modules, and takes the place of their own counts.

    The modules read it when their kernels run, so a recomputed forward pass (torch.utils.checkpoint) has
    the masks of the first one, and each replay of a captured step its own.  The program advances it after
    each step's backward pass, in the capture or between replays, with `counters[:, 1] += 1`; until then
    every call of a module has the same mask.  State dicts save and load it, in place."""
    modules = [m for m in model.modules() if isinstance(m, CountedMasks)]
    rows = [m.next_count(m.get_extra_state()) for m in modules]
    counters = torch.stack(rows) if rows else torch.zeros(0, 2, dtype=torch.int64)
    counters = counters.to(device)
    for m, row in zip(modules, counters):
        m.counter, m.counter_version = row, None
    return counters
