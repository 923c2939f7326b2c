"""Sampling as the reference's Sampler does it (src/sampler.cpp): argmax with the
lowest index on ties, temperature sampling by a walk along the running sum,
and the probability of one token.  The arithmetic runs in HIP kernels over the
float32 logits on the device.  Randomness is explicit: the uniform number of a
draw is a function of (seed, request id, step) alone, so a request's tokens do
not depend on what else is in its batch (the reference seeds the C library's
global generator with the wall clock, src/main.cpp:66, src/sampler.cpp:6-9)."""
import math

import torch

from ..ops import kernels

_MASK = (1 << 64) - 1


def _mix(x):
    x &= _MASK
    x = ((x ^ (x >> 30)) * 0xBF58476D1CE4E5B9) & _MASK
    x = ((x ^ (x >> 27)) * 0x94D049BB133111EB) & _MASK
    return x ^ (x >> 31)


def uniform(seed, request_id, step):
    """A number in [0, 1) with 24 random bits for draw `step` of request `request_id`."""
    h = _mix(_mix(_mix(seed * 0x9E3779B97F4A7C15 + 1) + request_id * 0xD1B54A32D192ED03 + 2) + step)
    return (h >> 40) / float(1 << 24)


class Drawn:
    """The tokens of one draw: on the device at once (`tokens`, int32 [R]), on the host once the
    copy that follows the sampling kernel has landed (`tolist()` waits for it, and for nothing
    that was queued later)."""

    def __init__(self, tokens, host, landed, sampler, turn):
        self.tokens = tokens
        self._host = host
        self._landed = landed
        self._sampler, self._turn = sampler, turn
        self._list = None

    def tolist(self):
        if self._list is None:
            if self._sampler._turn - self._turn >= Sampler.HOST_BUFFERS:
                raise RuntimeError("the tokens of a draw are read after %d later draws have taken its host buffer"
                                   % Sampler.HOST_BUFFERS)
            self._landed.synchronize()
            self._list = self._host.tolist()
        return self._list


def _of_rows(value):
    """Whether a setting is a sequence, one number a row (and no number of Python's, numpy's or torch's for all of them)."""
    return hasattr(value, "__len__") and getattr(value, "ndim", 1) > 0


# what each setting of a draw may be
SETTINGS = {"temperature": (0.0, math.inf), "top_k": (0, 2 ** 31 - 1), "top_p": (0.0, 1.0), "min_p": (0.0, 1.0)}


class Sampler:
    HOST_BUFFERS = 4          # draws whose host copies may be unread at the same time

    def __init__(self, seed=0):
        self.seed = int(seed)
        self._host = []           # pinned buffers and the events after the copies into them, used in turn
        self._turn = 0

    def _host_buffers(self, R):
        """The pinned pair of this turn: int32 for the tokens on their way back, float32 for the
        uniform numbers and the rows' settings on their way out, and the event behind the draw that used them last.
        A draw that fails behind this leaves the turn where it was, and the next one takes the same pair."""
        turn = self._turn % self.HOST_BUFFERS
        if turn == len(self._host):
            n = max(R, 64)
            self._host.append([torch.empty(n, dtype=torch.int32, pin_memory=True),
                               torch.empty(5 * n, dtype=torch.float32, pin_memory=True), torch.cuda.Event()])
            return self._host[-1]
        entry = self._host[turn]
        entry[2].synchronize()
        if entry[0].shape[0] < R:
            entry[0] = torch.empty(R, dtype=torch.int32, pin_memory=True)
            entry[1] = torch.empty(5 * R, dtype=torch.float32, pin_memory=True)
        return entry

    @staticmethod
    def _checked(settings, R):
        """The settings of a draw under filters, each a number for all rows or a list of one for each, after the checks."""
        out = {}
        for name, value in settings.items():
            of_rows = _of_rows(value)
            values = [int(v) if name == "top_k" else float(v) for v in (value if of_rows else [value])]
            if of_rows and len(values) != R:
                raise ValueError("%s: %d settings for %d rows" % (name, len(values), R))
            low, high = SETTINGS[name]
            if not all(low <= v <= high for v in values):
                raise ValueError("%s: %s is not between %s and %s" % (name, values, low, high))
            out[name] = values if of_rows else values[0]
        return out

    def _filtered(self, logits, out, host, settings, request_ids, steps):
        """sample_filtered with the rows' numbers and settings (_checked) uploaded together.  The workspace is the current stream's own memory
        until the draw has run (the allocator hands it on within the stream only): draws on several streams may run at the same time."""
        R, V = logits.shape
        rows = host[:5 * R].view(5, R)
        rows[0] = torch.tensor([uniform(self.seed, r, s) for r, s in zip(request_ids, steps)], dtype=torch.float32)
        for at, (name, value) in zip(rows[1:], settings.items()):
            dtype = torch.int32 if name == "top_k" else torch.float32
            at.view(dtype).copy_(torch.tensor(value, dtype=dtype))
        dev = torch.empty((5, R), dtype=torch.float32, device=logits.device)
        dev.copy_(rows, non_blocking=True)                # from pinned memory: the host does not wait for the queue
        workspace = torch.empty(kernels.sample_filtered_workspace(R, V), dtype=torch.int32, device=logits.device)
        kernels.sample_filtered(logits, dev[0], out, temperature=dev[1], top_k=dev[2].view(torch.int32), top_p=dev[3], min_p=dev[4],
                                workspace=workspace)

    def draw(self, logits, temperature, request_ids, steps, top_k=0, top_p=1.0, min_p=0.0):
        """One token for each row of logits [R, vocab] (device, float32); temperature 0 is argmax.  top_k (0: off), top_p (1: off) and
        min_p (0: off) leave a part of the tokens to draw from (kernels.sample_filtered); they and the temperature are numbers for all rows
        or sequences of one for each.  A refused draw changes nothing; draws may be queued on several streams, each behind what made its logits.
        Nothing waits for the device here: the tokens can feed the next step from where they lie
        while the host reads them a step later."""
        R = logits.shape[0]
        settings = {"temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p}
        filtered = any(_of_rows(v) for v in settings.values()) or (top_k, top_p, min_p) != (0, 1.0, 0.0)
        if filtered:
            settings = self._checked(settings, R)         # in front of the buffers: a refused draw takes none
        out = torch.empty(R, dtype=torch.int32, device=logits.device)
        host, host_u, landed = self._host_buffers(R)
        if filtered:
            self._filtered(logits, out, host_u, settings, request_ids, steps)
        elif temperature == 0.0:
            kernels.argmax(logits, out)
        else:
            host_u[:R] = torch.tensor([uniform(self.seed, r, s) for r, s in zip(request_ids, steps)],
                                      dtype=torch.float32)
            u = torch.empty(R, dtype=torch.float32, device=logits.device)
            u.copy_(host_u[:R], non_blocking=True)          # from pinned memory: the host does not wait for the queue
            kernels.sample(logits, u, float(temperature), out)
        host[:R].copy_(out, non_blocking=True)
        landed.record(torch.cuda.current_stream(out.device.index))
        self._turn += 1
        return Drawn(out, host[:R], landed, self, self._turn)

    def sample(self, logits, temperature, request_ids, steps, **filters):
        """As draw, but returns the tokens as a list of ints."""
        return self.draw(logits, temperature, request_ids, steps, **filters).tolist()

    def argmax(self, logits):
        out = torch.empty(logits.shape[0], dtype=torch.int32, device=logits.device)
        kernels.argmax(logits, out)
        return out.tolist()

    def prob(self, logits, index):
        """softmax(logits[r])[index[r]] at temperature 1 (src/sampler.cpp:11-25)."""
        idx = torch.tensor(list(index), dtype=torch.int32, device=logits.device)
        out = torch.empty(logits.shape[0], dtype=torch.float32, device=logits.device)
        kernels.token_prob(logits, idx, out)
        return out.tolist()


def filters_for_all(top_k, top_p, min_p):
    """What a loop whose batches shrink hands to every draw: one number for all requests each, checked before the first step ({}: all are off)."""
    settings = {"top_k": top_k, "top_p": top_p, "min_p": min_p}
    for name, value in settings.items():
        one_for_all(name, value)
    settings = Sampler._checked(settings, 0)
    return {} if tuple(settings.values()) == (0, 1.0, 0.0) else settings


def one_for_all(name, value):
    if _of_rows(value):
        raise ValueError("%s: a generation loop takes one number for all requests (Sampler.draw takes one for each row)" % name)
