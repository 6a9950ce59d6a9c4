"""Step tables, beam selection and beam reordering through the native call path and through Python: the same bits, the same refusals."""
import threading

import pytest
import torch

import wuda_b200 as wuda
from wuda_b200 import ops

pytestmark = pytest.mark.gpu


class Off:
    def __getattr__(self, name):
        return lambda *a: None


class Recorder:
    def __init__(self, native):
        self.native, self.took = native, []

    def __getattr__(self, name):
        f = getattr(self.native, name)

        def call(*args):
            done = f(*args)
            self.took.append((name, done is not None))
            return done
        return call


def _world(seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    lengths = i32(300, 7, 1000, 255, 64)
    page = lambda n: torch.arange(n * 5, dtype=torch.int32, device="cuda").view(5, n).contiguous()
    plan = wuda.StepTables(lengths, page(6), page(6) + 40, page(1), torch.arange(50, 60, dtype=torch.int32, device="cuda"),
                           torch.arange(80, 90, dtype=torch.int32, device="cuda"), i32(10, 9), max_rows=5, max_tokens=20)
    state = torch.randn(5, 12, generator=g, device="cuda")
    pool = torch.randint(0, 256, (30, 64 * 132), generator=g, device="cuda", dtype=torch.uint8)
    again = lengths.clone().fill_(300)
    reorder = wuda.BeamReorder(again, 2, states=[state], pools=[wuda.PagedState(pool, page(6), 64, (128, 4), tokens_per_entry=4)])
    logits = torch.randn(2, 3, 501, generator=g, device="cuda")
    scores = torch.randn(2, 3, generator=g, device="cuda")
    done = torch.tensor([[0, 1, 0], [0, 0, 0]], device="cuda") > 0
    return plan, reorder, logits, scores, done, i32


def _run():
    plan, reorder, logits, scores, done, i32 = _world()
    out = []
    for new in (None, i32(3, 0, 5)):
        plan.step(i32(2, 0, 4), new)
        out += [t.clone() for t in plan.out.values()] + [plan.lengths.clone(), plan.free_counts.clone(), plan.idx_table.clone()]
    slots = torch.empty(2, 2, dtype=torch.int32, device="cuda")
    reorder.run(i32(0, 0, 1, 0).view(2, 2), i32(3, 1, 4, 0).view(2, 2), slots)
    out += [slots, reorder.states[0], reorder.pools[0].data]
    for kind in (torch.float32, torch.bfloat16, torch.float16):
        for call in (lambda x: wuda.beam_select(x, scores), lambda x: wuda.beam_select(x, scores, 7, finished=done, eos_token=5),
                     lambda x: wuda.beam_select(x[:, :, 1:], scores, 2, eos_token=499)):
            out += list(call(logits.to(kind)))
    torch.cuda.synchronize()
    return out


def test_both_ways_give_the_same_bits(monkeypatch):
    _run()                                   # (the scratch exists from here on)
    recorder = Recorder(ops._fast)
    monkeypatch.setattr(ops, "_fast", recorder)
    native = _run()
    assert recorder.took and all(took for _, took in recorder.took) and {n for n, _ in recorder.took} == {"step_tables", "beam_reorder", "beam_select"}
    monkeypatch.setattr(ops, "_fast", Off())
    for a, b in zip(native, _run()):
        assert a.dtype == b.dtype and torch.equal(a, b)


@pytest.mark.parametrize("way", ["native", "python"])
def test_both_ways_refuse_the_same(way, monkeypatch):
    if way == "python":
        monkeypatch.setattr(ops, "_fast", Off())
    plan, reorder, logits, scores, done, i32 = _world()
    four = i32(0, 1, 2, 3)
    for call in (lambda: plan.step(i32(0, 1, 2, 3, 4, 0)), lambda: plan.step(four.long()), lambda: plan.step(four, four[:2]), lambda: plan.step(four.cpu()),
                 lambda: plan.step(i32(0, 1, 2, 3)[::2]), lambda: reorder.run(i32(0, 0, 0), i32(0, 1, 2), i32(0, 0, 0)),
                 lambda: reorder.run(four, four, four), lambda: reorder.run(four, four.long(), four), lambda: reorder.run(four, i32(0, 1), i32(0, 1)),
                 lambda: wuda.beam_select(logits, scores, 65), lambda: wuda.beam_select(logits, scores, 0), lambda: wuda.beam_select(logits, scores, eos_token=501),
                 lambda: wuda.beam_select(logits, scores, eos_token=-1), lambda: wuda.beam_select(logits, scores, finished=done),
                 lambda: wuda.beam_select(logits, scores[:1]), lambda: wuda.beam_select(logits.int(), scores)):
        with pytest.raises(wuda.WudaError):
            call()


def test_threads_on_streams_of_their_own():
    """Selections of different sizes from eight threads at once, each on its own stream: scratch and counters are per stream."""
    cases = []
    for i in range(8):
        g = torch.Generator(device="cuda").manual_seed(i)
        x, s = torch.randn(1 + i, 4, 5000 * (i + 1), generator=g, device="cuda").bfloat16(), torch.randn(1 + i, 4, generator=g, device="cuda")
        cases.append((x, s, [t.clone() for t in wuda.beam_select(x, s, 8)]))
    torch.cuda.synchronize()
    wrong = []

    def work(x, s, want):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(40):
                got = wuda.beam_select(x, s, 8)
            stream.synchronize()
            wrong.append(not all(torch.equal(a, b) for a, b in zip(got, want)))
    threads = [threading.Thread(target=work, args=c) for c in cases]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert wrong == [False] * 8
