"""When the language model makes its 4-bit copies of the weights anew, and into which memory: on the host, with a quantisation
that keeps the weights' numbers and a GPU that notes what it is asked."""

from __future__ import annotations

import copy
import pickle
import threading

import pytest
import torch
from torch import nn

from mamba3_amd import KulaMambaLM, MXTensor, block


def kept_numbers(w, format="e2m1"):
    rows, k = w.shape
    data = torch.zeros(rows, -(-k // 128) * 64, dtype=torch.uint8)
    data[:, :k] = w[:, :data.shape[1]].to(torch.uint8)
    return MXTensor(data, torch.full((rows, -(-k // 128) * 4), 127, dtype=torch.uint8), (rows, k), format)


class Gpu:
    """What _mx_copy asks of torch.cuda."""

    def __init__(self):
        self.asked, self.capturing, self.stream, self.on_wait = [], False, 0, lambda: None

    def current_stream(self, device=None):
        return self

    def synchronize(self, device=None):
        self.asked.append("wait" if device is None else "wait for all")
        self.on_wait()

    def is_current_stream_capturing(self):
        return self.capturing


@pytest.fixture
def gpu(monkeypatch):
    gpu = Gpu()
    monkeypatch.setattr(block, "quantize_mx", kept_numbers)
    for name in ("current_stream", "synchronize", "is_current_stream_capturing"):
        monkeypatch.setattr(torch.cuda, name, getattr(gpu, name))
    monkeypatch.setattr(block._native, "stream_of", lambda t: gpu.stream)
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, stream: gpu.asked.append(("reads", t.data_ptr(), gpu.stream)))
    return gpu


def linear(start=0, rows=3, k=20):
    lin = nn.Linear(k, rows, bias=False)
    with torch.no_grad():
        lin.weight.copy_((torch.arange(rows * k) + start).view(rows, k))
    return lin


def get(lin):
    return block._mx_copy(lin, lin.weight)


def fresh(lin):
    return torch.equal(get(lin).data, kept_numbers(lin.weight.detach()).data)


@torch.no_grad()
def test_a_copy_follows_a_new_parameter_of_the_same_memory(gpu):
    """It counts its versions anew, so that address and version are the old parameter's while the numbers are others."""
    lin = linear()
    assert fresh(lin)
    old = lin.weight
    lin.weight = nn.Parameter(old.data)
    assert lin.weight._version < old._version and lin.weight.data_ptr() == old.data_ptr()
    while lin.weight._version < old._version:
        lin.weight.add_(1.0)
    assert fresh(lin)
    lin.weight.add_(1.0)
    assert fresh(lin)


@torch.no_grad()
def test_a_copied_or_pickled_module_makes_its_own(gpu):
    lin = linear()
    mine = get(lin)
    for other in (copy.deepcopy(lin), pickle.loads(pickle.dumps(lin))):
        assert fresh(other) and get(other).data.data_ptr() != mine.data.data_ptr()
        other.weight.add_(5.0)
        assert fresh(other) and fresh(lin) and get(lin) is mine


@torch.no_grad()
def test_a_copy_is_made_once(gpu):
    lin = linear()
    first = get(lin)
    waits = len(gpu.asked)
    assert all(get(lin) is first for _ in range(3)) and len(gpu.asked) == waits
    lin.to(torch.bfloat16)
    assert fresh(lin)


def test_weights_that_do_not_count_their_changes_are_refused(gpu):
    with torch.inference_mode():
        made = linear()
        with pytest.raises(RuntimeError, match="inference_mode"):
            get(made)
    with pytest.raises(RuntimeError, match="inference_mode"):
        get(made)
    lin = linear()
    first = get(lin)
    with torch.inference_mode():  # the mode itself is no matter: other parameters count their changes in it
        assert get(lin) is first
        lin.weight.add_(3.0)
        assert fresh(lin)
        lin.weight = nn.Parameter(lin.weight + 1)
        with pytest.raises(RuntimeError, match="inference_mode"):
            get(lin)


def copies(lm):
    return [m.__dict__["_mx"].mx for m in lm.modules() if "_mx" in m.__dict__]


def small_lm(**kw):
    return KulaMambaLM(50, 64, n_layers=2, d_state=16, headdim=16, mimo_rank=1, **kw)


@torch.no_grad()
def test_quantising_again_makes_the_copies_anew_in_their_memory(gpu):
    """Graphs that were captured with them read it."""
    lm = small_lm().quantize_mx()
    gpu.capturing = True
    lm._mx_head(), [layer._mx_projections() for layer in lm.layers]
    gpu.capturing = False
    at = [(c.data.data_ptr(), c.scales.data_ptr()) for c in copies(lm)]
    assert len(at) == 9  # four a block and the head's
    for p in lm.parameters():
        p.data.fill_(7.0)  # leaves no trace
    assert lm.quantize_mx() is lm
    assert [(c.data.data_ptr(), c.scales.data_ptr()) for c in copies(lm)] == at
    assert all((c.data[:, 0] == 7).all() for c in copies(lm))
    assert not copies(lm.quantize_mx(False)) and not lm.mx_weights and not lm.layers[1].mx_weights


@torch.no_grad()
def test_a_call_that_fails_leaves_the_model_as_it_was(gpu):
    lm = small_lm().quantize_mx()
    mine = [lm._mx_head()]
    hook = lm.lm_head.register_forward_hook(lambda *a: None)
    with pytest.raises(RuntimeError, match="hooks"):
        lm.quantize_mx()
    hook.remove()
    assert lm.mx_weights and lm.layers[0].mx_weights and len(copies(lm)) == 9 and mine[0] in copies(lm)
    biased = small_lm(bias=True)
    with pytest.raises(RuntimeError, match="bias"):
        biased.quantize_mx()
    assert not biased.mx_weights and not copies(biased)


@torch.no_grad()
def test_a_new_copy_leaves_the_old_one_to_work_under_way(gpu):
    lin = linear()
    mine = get(lin)
    numbers = mine.data.clone()
    other = nn.Parameter(lin.weight + 9.0)
    for change in (lambda: lin.weight.add_(1.0), lambda: setattr(lin, "weight", other)):
        change()
        assert fresh(lin) and get(lin) is not mine and torch.equal(mine.data, numbers)
    mine = get(lin)
    numbers = mine.data.clone()
    assert block._mx_copy(lin, lin.weight, anew=True) is not mine and torch.equal(mine.data, numbers)


@torch.no_grad()
def test_a_copy_that_a_graph_reads_is_overwritten_behind_all_work(gpu):
    lin = linear()
    get(lin)
    gpu.capturing = True
    mine = get(lin)
    gpu.capturing = False
    for i in range(3):
        lin.weight.add_(1.0)
        numbers, seen = mine.data.clone(), []
        gpu.on_wait = lambda: seen.append((gpu.asked[-1], torch.equal(mine.data, numbers)))
        assert get(lin) is mine and not torch.equal(mine.data, numbers) and fresh(lin)
        assert seen == [("wait for all", True), ("wait", False)]


@torch.no_grad()
def test_the_allocator_learns_each_stream_that_reads_a_copy(gpu):
    lin = linear()
    mine = get(lin)
    assert not [a for a in gpu.asked if a[0] == "reads"]  # the stream it was made on it knows
    for gpu.stream in (0, 5, 5, 6, 0, 5):
        get(lin)
    want = [("reads", t.data_ptr(), stream) for stream in (5, 6) for t in (mine.data, mine.scales)]
    assert [a for a in gpu.asked if a[0] == "reads"] == want


@torch.no_grad()
def test_threads_that_find_a_copy_stale_make_it_once(gpu, monkeypatch):
    lin, made, meet = linear(), [], threading.Barrier(4)

    def slow(w, format="e2m1"):
        made.append(threading.get_ident())
        threading.Event().wait(0.05)
        return kept_numbers(w, format)

    monkeypatch.setattr(block, "quantize_mx", slow)
    got = [None] * 4

    def one(i):
        with torch.no_grad():
            meet.wait()
            got[i] = get(lin)

    for turn in range(2):
        threads = [threading.Thread(target=one, args=(i,)) for i in range(4)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert len(made) == turn + 1 and all(g is got[0] for g in got) and fresh(lin)
        lin.weight.add_(1.0)


@torch.no_grad()
def test_a_change_while_a_copy_is_made_is_not_missed(gpu, monkeypatch):
    lin = linear()

    def changed_meanwhile(w, format="e2m1"):
        numbers = kept_numbers(w, format)
        lin.weight.add_(1.0)
        return numbers

    monkeypatch.setattr(block, "quantize_mx", changed_meanwhile)
    get(lin)
    monkeypatch.setattr(block, "quantize_mx", kept_numbers)
    assert fresh(lin)


@torch.no_grad()
def test_readers_of_a_copy_that_a_graph_reads_too_are_known(gpu):
    lin = linear()
    mine = get(lin)
    gpu.stream, gpu.capturing = 3, True
    get(lin)
    gpu.capturing = False
    gpu.asked.clear()
    for turn in range(2):
        for gpu.stream in (0, 5, 3, 5):
            assert get(lin) is mine
        lin.weight.add_(1.0)
    gpu.stream = 9  # makes the copy anew in the graph's memory, and reads it
    assert get(lin) is mine
    reads = [a for a in gpu.asked if a[0] == "reads"]
    assert reads == [("reads", t.data_ptr(), stream) for stream in (5, 3, 9) for t in (mine.data, mine.scales)]


@torch.no_grad()
def test_memory_that_a_graph_reads_is_given_back_behind_all_work(gpu):
    lm = small_lm().quantize_mx()
    gpu.asked.clear()
    lm.quantize_mx(False).quantize_mx()
    assert "wait for all" not in gpu.asked  # the allocator knows the other readers
    gpu.capturing = True
    lm._mx_head()
    gpu.capturing = False
    gpu.asked.clear()
    lm.quantize_mx(False)
    assert gpu.asked == ["wait for all"] and not copies(lm)
    lin = linear()
    get(lin)
    gpu.capturing = True
    old = get(lin)
    gpu.capturing = False
    gpu.asked.clear()
    lin.weight = nn.Parameter(torch.ones(5, 40))  # no room for it in the old one's memory
    assert get(lin) is not old and gpu.asked == ["wait for all", "wait"] and fresh(lin)
