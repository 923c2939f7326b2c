"""The sampler's buffers without a GPU: stand-ins for its kernels write each draw's own number, pinned memory and events are plain ones."""
import numpy as np
import pytest
import torch

from yalm_amd.sampling import Sampler, sampler as module


class Event:
    def synchronize(self):
        pass

    def record(self, stream=None):
        pass


@pytest.fixture
def stand_in(monkeypatch):
    """The draws' number, and the workspaces that they were given."""
    seen = {"draws": 0, "workspaces": [], "fail": False}
    plain = torch.empty

    def empty(*shape, pin_memory=False, **kw):
        return plain(*shape, **kw)

    def draw(logits, out):
        if seen["fail"]:
            raise RuntimeError("no launch")
        out.fill_(seen["draws"])
        seen["draws"] += 1

    def sample_filtered(logits, u, out, workspace=None, **kw):
        seen["workspaces"].append(workspace)
        draw(logits, out)

    monkeypatch.setattr(module.torch, "empty", empty)
    monkeypatch.setattr(module.torch.cuda, "Event", Event)
    monkeypatch.setattr(module.torch.cuda, "current_stream", lambda *a: None)
    monkeypatch.setattr(module.kernels, "argmax", draw)
    monkeypatch.setattr(module.kernels, "sample", lambda logits, u, t, out: draw(logits, out))
    monkeypatch.setattr(module.kernels, "sample_filtered", sample_filtered)
    monkeypatch.setattr(module.kernels, "sample_filtered_workspace", lambda R, V: 12)
    return seen


def read_late(sampler, how, n=8):
    """n draws, each read only when no more may be unread."""
    logits, got, waiting = torch.zeros((2, 5)), [], []
    for i in range(n):
        waiting.append(sampler.draw(logits, how.get("temperature", 0.7), [0, 1], [i, i], **{k: v for k, v in how.items() if k != "temperature"}))
        if len(waiting) == Sampler.HOST_BUFFERS:
            got.append(waiting.pop(0).tolist())
    return got + [d.tolist() for d in waiting]


HOW = [{"temperature": 0.0}, {}, {"top_p": 0.9}, {"temperature": [0.0, 0.5], "top_k": 3}]


REFUSED = [{"top_p": 1.5}, {"min_p": -0.1}, {"top_k": [1, 2, 3]}, {"top_k": -1}, {"top_p": float("nan")}, {"temperature": -1.0, "top_k": 3}]


@pytest.mark.parametrize("before,refusals", [(0, 1), (0, 3), (1, 1), (3, 1), (2, 2), (4, 1), (6, 5)])
@pytest.mark.parametrize("how", HOW)
def test_draws_behind_refused_ones_are_their_own(stand_in, how, before, refusals):
    """However many draws came before them, refused ones move no buffer that a draw behind them uses."""
    s = Sampler(3)
    assert read_late(s, how, before) == [[i, i] for i in range(before)]
    for bad in (REFUSED * 2)[before:before + refusals]:
        with pytest.raises(ValueError, match=next(iter(bad))):
            s.draw(torch.zeros((2, 5)), request_ids=[0, 1], steps=[0, 0], **{"temperature": 0.7, **bad})
    assert read_late(s, how) == [[before + i] * 2 for i in range(8)]


@pytest.mark.parametrize("how", HOW)
def test_draws_behind_a_failed_one_are_their_own(stand_in, how):
    """A launch that fails leaves the buffers in turn, too."""
    s = Sampler(3)
    for before in (0, 8, 16):
        stand_in["fail"] = True
        with pytest.raises(RuntimeError, match="no launch"):
            read_late(s, how)
        stand_in["fail"] = False
        assert read_late(s, how) == [[before + i] * 2 for i in range(8)]


def test_draws_under_filters_have_workspaces_of_their_own(stand_in):
    """Draws on several streams may run at the same time: as long as one's workspace lives, no other draw is given it."""
    s = Sampler(3)
    draws = [s.draw(torch.zeros((2, 5)), 0.7, [0, 1], [i, i], top_p=0.9) for i in range(3)]
    assert len({w.data_ptr() for w in stand_in["workspaces"]}) == 3 and all(w.numel() >= 12 for w in stand_in["workspaces"])
    assert [d.tolist() for d in draws] == [[i, i] for i in range(3)]


class NoEngine:
    """An engine that a refused call never touches."""
    n_positions, max_draft, max_draft_depth = 64, 8, 8

    def __getattr__(self, name):
        raise AssertionError("the engine's %s was asked for" % name)


@pytest.mark.parametrize("loop", ["generate", "generate_drafted"])
@pytest.mark.parametrize("name,value", [("top_k", [3, 5]), ("top_k", np.array([3, 5])), ("top_p", torch.tensor([0.5, 0.9])), ("min_p", (0.1, 0.1)), ("temperature", [0.7, 0.8]),
                                        ("temperature", np.full(2, 0.5)), ("top_k", -1), ("top_p", 1.5), ("min_p", float("nan"))])
def test_loops_take_one_number_for_all_requests(loop, name, value):
    """Refused before the first step, where a sequence failed once the first request had left its batch, and the others' tokens with it."""
    import yalm_amd
    with pytest.raises(ValueError, match=name):
        getattr(yalm_amd, loop)(NoEngine(), [[1, 2], [3]], stop_ids=[], max_new_tokens=4, sampler=Sampler(1), **{name: value})


def test_a_loop_s_numbers_of_any_kind():
    from yalm_amd.sampling.sampler import filters_for_all
    assert filters_for_all(0, 1.0, 0.0) == filters_for_all(np.int64(0), np.float32(1), torch.tensor(0.0)) == filters_for_all(0, 1, 0) == {}
    assert filters_for_all(np.array(7), torch.tensor(0.5), 0) == {"top_k": 7, "top_p": 0.5, "min_p": 0.0}
