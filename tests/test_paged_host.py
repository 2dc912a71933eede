"""paged.PagedEngine's bookkeeping without a GPU: a model without layers, stand-ins for the kernels and for CUDA graphs. The
"model" answers each sequence with its last token plus one, and a write of a row is recorded as (sequence's page, slot)."""
from contextlib import contextmanager

import pytest
import torch

import model as M
import paged

VOCAB = 256


class Ops:
    error = 0

    def set_pdl(self, on):
        pass

    def attention_workspace(self, device):
        return torch.zeros(64, dtype=torch.uint8)

    def gemm_scratch(self, device, rows, shapes):
        return torch.zeros(64, dtype=torch.uint8)

    def finalize(self, best, token, out_tokens, state):
        nxt = 0xFFFFFFFF - (best & 0xFFFFFFFF)
        token.copy_(nxt)
        out_tokens[torch.arange(len(nxt)), state[:, 1].long()] = nxt.to(torch.int32)
        state += 1

    def device_error(self):
        e, self.error = self.error, 0
        return e


class Engine(paged.PagedEngine):
    """Records what each pass writes: (page, slot) of every new row, by the arguments that the kernels get."""

    def _forward(self, tokens, cu, lens, table, max_q, whole, last):
        self.passes = getattr(self, "passes", 0) + 1
        self.batches = getattr(self, "batches", []) + [(cu[1:] - cu[:-1]).tolist()]
        P = self.page_size
        for b in range(len(lens)):
            n = int(cu[b + 1] - cu[b])
            for i in range(n):
                pos = int(lens[b]) - n + i
                page = int(table[b, pos // P]) if pos // P < table.shape[1] else -1
                if not 0 <= page < self.pages:
                    self.k.error = 2
                else:
                    self.written.append((page, pos % P))
            self.best[b] = 0xFFFFFFFF - (int(tokens[cu[b + 1] - 1]) + 1) % VOCAB


class Graph:
    recording = None

    def replay(self):
        self.body()


@pytest.fixture(scope="module")
def model():
    return M.Qwen3FP8Decode.synthetic(M.Config(vocab=VOCAB), max_seq=64, device="cpu", n_layers=0)


@pytest.fixture
def make(model, monkeypatch):
    """make(pages, ...): an engine on the CPU."""
    ops = Ops()
    monkeypatch.setattr(paged, "ops", lambda: ops)

    class Stream:
        def wait_stream(self, other):
            pass

    @contextmanager
    def on(stream):
        yield

    monkeypatch.setattr(torch.cuda, "Stream", Stream)
    monkeypatch.setattr(torch.cuda, "current_stream", Stream)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda: None)
    monkeypatch.setattr(torch.cuda, "stream", on)
    monkeypatch.setattr(torch.cuda, "CUDAGraph", Graph)

    def build(pages, **kw):
        kw = {**dict(page_size=16, max_rows=64, max_seqs=8), **kw}
        eng = Engine(model, pages, **kw)
        eng.pages, eng.written, eng.k.error = pages, [], 0

        @contextmanager
        def capture(graph):
            """The body of the capture, run again by a replay. (The recording run's own effects are undone.)"""
            keep = [t.clone() for t in (eng.token, eng.state, eng.out_tokens)]
            written, batches = list(eng.written), list(eng.batches)
            yield
            for t, old in zip((eng.token, eng.state, eng.out_tokens), keep):
                t.copy_(old)
            eng.written, eng.batches = written, batches

            def body():
                torch.add(eng.state[:, 0], 1, out=eng.g_lens)
                eng._forward(eng.token, eng.g_cu, eng.g_lens, eng.g_table, 1, False, None)
                eng.k.finalize(eng.best[:len(eng.g_lens)], eng.token, eng.out_tokens, eng.state)
            graph.body = body
        monkeypatch.setattr(torch.cuda, "graph", capture)
        return eng
    return build


def captured(eng, prompts=((1, 2, 3), (50,)), steps=4):
    seqs = [eng.new() for _ in prompts]
    toks = eng.step(list(zip(seqs, prompts)))
    eng.capture(seqs, toks, steps)
    return seqs, toks


def test_decode_goes_on_from_the_capture(make):
    eng = make(8)
    seqs, toks = captured(eng)
    assert toks == [4, 51]
    assert eng.decode(2) == [[5, 6], [52, 53]] and eng.decode(2) == [[7, 8], [54, 55]]
    assert [eng.lens[s] for s in seqs] == [7, 5]


def test_decode_refuses_a_sequence_that_was_released(make):
    """Its pages may be another's by then: nothing is replayed."""
    eng = make(4)
    (a, b), _ = captured(eng)
    eng.decode(1)
    eng.release(a)
    other = eng.new()
    eng.step([(other, [9] * 40)])                    # takes the released page too
    written, lens = list(eng.written), dict(eng.lens)
    with pytest.raises(ValueError, match="capture"):
        eng.decode(1)
    assert eng.written == written and eng.lens == lens


def test_decode_refuses_a_sequence_that_went_on(make):
    """A pass on a captured sequence leaves the graph's position behind it."""
    eng = make(8)
    (a, b), _ = captured(eng)
    eng.decode(1)
    nxt = eng.step([(b, [70])])
    assert nxt == [71]
    written, lens = list(eng.written), dict(eng.lens)
    with pytest.raises(ValueError, match="capture"):
        eng.decode(1)
    assert eng.written == written and eng.lens == lens
    eng.capture([a, b], [6, 71], 2)                  # a new capture goes on from there
    assert eng.decode(2) == [[7, 8], [72, 73]]


def test_decode_refuses_before_a_capture_and_steps_that_are_none(make):
    eng = make(8)
    with pytest.raises(ValueError, match="capture"):
        eng.decode(1)
    seqs, _ = captured(eng)
    before = dict(eng.lens)
    for n in (-1, 5):
        with pytest.raises(ValueError):
            eng.decode(n)
    assert eng.lens == before and eng.decode(0) == [[], []]


def test_a_table_names_no_page_past_a_sequences_own(make):
    """Entries past the reservation are -1, which the kernels refuse, not page 0, which may be another sequence's."""
    eng = make(8, max_len=64)
    s = eng.new()
    eng.reserve(s, 17)
    table = eng._table([s])
    assert table.tolist() == [eng.tables[s] + [-1, -1]]


@pytest.mark.parametrize("bad", ["no steps", "negative steps", "one sequence twice", "a token short", "a token over"])
def test_capture_refuses(make, bad):
    """Nothing is written and no page taken: the warm-up step needs a reserved position, and a row a token."""
    eng = make(8)
    seqs = [eng.new(), eng.new()]
    toks = eng.step([(seqs[0], [1] * 16), (seqs[1], [2] * 16)])      # both end with their page
    args = {"no steps": (seqs, toks, 0), "negative steps": (seqs, toks, -1), "one sequence twice": (seqs[:1] * 2, toks, 2),
            "a token short": (seqs, toks[:1], 2), "a token over": (seqs, toks + [1], 2)}[bad]
    free, written = list(eng.free), list(eng.written)
    with pytest.raises(ValueError):
        eng.capture(*args)
    assert eng.free == free and eng.written == written and eng.k.error == 0


def test_capture_takes_no_pages_where_the_pool_has_too_few(make):
    eng = make(3)
    seqs = [eng.new(), eng.new()]
    toks = eng.step([(seqs[0], [1] * 16), (seqs[1], [2] * 16)])
    with pytest.raises(RuntimeError, match="out of pages"):
        eng.capture(seqs, toks, 4)                   # a page each: one is left
    assert len(eng.free) == 1


def test_a_pass_takes_no_pages_where_the_pool_has_too_few(make):
    eng = make(3)
    a, b = eng.new(), eng.new()
    with pytest.raises(RuntimeError, match="out of pages"):
        eng.step([(a, [1] * 16), (b, [1] * 33)])
    assert len(eng.free) == 3 and eng.lens == {a: 0, b: 0} and eng.step([(b, [1] * 33)]) == [2]


@pytest.mark.parametrize("bad", ["empty prompt", "too long", "a failing pass"])
def test_generate_gives_its_pages_back_when_it_fails(make, bad):
    eng = make(8, max_len=48)
    kept = eng.new()
    eng.step([(kept, [3])])
    prompts = [[1, 2], list(range(20))]
    if bad == "empty prompt":
        prompts.append([])
    elif bad == "too long":
        prompts.append([1] * 47)
    else:
        step = eng.step
        eng.step = lambda batch: step(batch) if eng.passes < 3 else (_ for _ in ()).throw(RuntimeError("pass failed"))
    with pytest.raises(ValueError if bad == "empty prompt" else RuntimeError):
        eng.generate(prompts, 4)
    assert len(eng.free) == 7 and list(eng.lens) == [kept]
    if bad != "a failing pass":
        assert eng.passes == 1                       # refused before anything ran


def test_generate_serves_in_turn_what_does_not_fit_together(make):
    """Finished sequences give their pages to those that wait; a prompt waits until its whole length has pages."""
    eng = make(4, max_len=64)
    prompts = [[10 * i + 1] * (17 + i) for i in range(5)]            # two pages each, with four new tokens
    assert eng.generate(prompts, 4) == [[10 * i + 1 + j for j in range(1, 5)] for i in range(5)]
    assert len(eng.free) == 4 and not eng.lens
    assert max(len(b) for b in eng.batches) == 2
    with pytest.raises(RuntimeError, match="out of pages"):
        make(3, max_len=64).generate(prompts + [[1] * 50], 4)
    kept = eng.new()
    eng.step([(kept, [5] * 33)])
    with pytest.raises(RuntimeError, match="out of pages"):          # one page is left, and nothing to wait for
        eng.generate(prompts[:1], 4)
    assert len(eng.free) == 1 and list(eng.lens) == [kept]


def test_generate_admits_everything_that_fits_at_once(make):
    """As many sequences as there is room for begin together, in the order they came."""
    eng = make(16, max_rows=40)
    prompts = [[1] * 30, [2] * 25, [3]]
    assert eng.generate(prompts, 3, chunk=16) == [[2, 3, 4], [3, 4, 5], [4, 5, 6]]
    assert eng.batches[:3] == [[16, 16, 1], [1, 14, 9], [1, 1, 1]]


def test_recover_resets_every_counter_of_a_pass(make):
    """A wait that gave up leaves the counters of the attention or of the linears mid-count."""
    eng = make(4)
    eng.ws.fill_(1)
    eng.linear_ws.fill_(1)
    eng.k.error = 1
    eng.recover()
    assert not eng.ws.any() and not eng.linear_ws.any()
    eng.check()


def test_a_pass_that_was_not_launched_leaves_the_lengths(make):
    """A refusal on the host (a table, a shape) wrote no rows: the sequences go on from where they were."""
    eng = make(4)
    s = eng.new()
    eng.step([(s, [1, 2])])
    forward, eng._forward = eng._forward, lambda *a: (_ for _ in ()).throw(RuntimeError("refused"))
    with pytest.raises(RuntimeError, match="refused"):
        eng.step([(s, [3])])
    eng._forward = forward
    assert eng.lens[s] == 2 and eng.step([(s, [3])]) == [4]


def test_export_refuses_a_cache_that_cannot_hold_the_sequence(make):
    eng = make(4)
    s = eng.new()
    eng.step([(s, [1] * 20)])
    cache = torch.zeros(0, 8, 64, 128, dtype=torch.bfloat16)
    eng.export(s, cache, cache.clone())
    for bad in (cache[:, :, :19], cache[:, :4], torch.zeros(1, 8, 64, 128, dtype=torch.bfloat16), cache[..., :64]):
        for k, v in ((bad, cache), (cache, bad)):
            with pytest.raises(ValueError, match="export"):
                eng.export(s, k, v)


def test_generate_takes_prompts_of_any_kind_once(make):
    eng = make(8)
    prompts = [range(5), (7, 8), iter([20, 30])]
    assert eng.generate(prompts, 2) == [[5, 6], [9, 10], [31, 32]]
    kept = [[1, 2], [3]]
    eng.generate(kept, 2)
    assert kept == [[1, 2], [3]]
