"""Beam search through PagedEngine on the GPU (a 2-layer model): what each step selects is checked against 64 bits, the result is
followed from the recorded steps by a beam search written apart, and the logits of every hypothesis are those of a pass over its
tokens alone, but for the order of sums (as for the paged engine's other tests: 0.1 of their norm, 0.25 over an e4m3 cache)."""
import math

import pytest
import torch

import model as M
from test_sharing_gpu import check_select

pytestmark = pytest.mark.gpu
PROMPTS = [[5, 17, 388, 3], [(7 * i) % 512 for i in range(150)], [400]]


def engine(vocab=512, **kw):
    from paged import PagedEngine
    m = M.Qwen3FP8Decode.synthetic(M.Config(layers=2, vocab=vocab), max_seq=512, seed=4, norm_init="random")
    return PagedEngine(m, **{**dict(pages=200, page_size=16, max_rows=64), **kw})


class Record:
    """The engine's ops with every beam_select's inputs and outputs kept (step by step, without graphs)."""

    def __init__(self, eng, monkeypatch):
        self.calls = []
        real = eng.k.beam_select

        def keep(logits, scores, cu, *out, workspace=None):
            real(logits, scores, cu, *out, workspace=workspace)
            self.calls.append((logits.clone(), scores.clone(), cu.tolist(), [t.tolist() for t in out]))

        monkeypatch.setattr(eng.k, "beam_select", keep)
        monkeypatch.setattr(eng, "beam_graph", False)


def search(calls, beams, eos, alpha, gen_len):
    """Beam search over the recorded candidates: [(ids, score, [(step, row) whose logits gave each id])] per prompt."""
    N = len(calls[0][2]) - 1
    out = []
    for b in range(N):
        live, ended = [([], 0.0, [], b)], []
        for t, (_, _, cu, (s, p, v)) in enumerate(calls):
            nxt, new = [], []
            for i in range(2 * beams):
                if p[b][i] < 0:
                    continue
                ids, _, rows, _ = live[p[b][i] - cu[b]]
                h = (ids + [v[b][i]], s[b][i], rows + [(t, p[b][i])])
                if v[b][i] == eos:
                    if i < beams:
                        new.append((h[0], h[1] / len(h[0]) ** alpha, h[2]))
                elif len(nxt) < beams:
                    nxt.append((*h, 0))
            ended = sorted(ended + new, key=lambda h: -h[1])[:beams]
            live = nxt
        both = ended + [(ids, s / len(ids) ** alpha, rows) for ids, s, rows, _ in live]
        out.append(sorted(both, key=lambda h: -h[1])[:beams])
    return out


@pytest.mark.parametrize("kv,beams,alpha,eos", [("bf16", 4, 1.0, None), ("bf16", 3, 0.6, "often"), ("fp8", 2, 0.0, "often"), ("bf16", 1, 1.0, None),
                                                ("bf16", 16, 1.0, "often")])
def test_beam_search(kv, beams, alpha, eos, monkeypatch):
    eng = engine(kv_dtype=kv, pages=1200 if beams == 16 else 200)
    steps = 12
    if eos == "often":      # a token that the first prompt's candidates hold
        s = eng.new()
        eng.step([(s, PROMPTS[0])])
        eos = int(eng.logits[0].float().topk(2).indices[1])
        eng.release(s)
    free = sorted(eng.free)
    rec = Record(eng, monkeypatch)
    got = eng.beam_search(PROMPTS, beams, steps, eos=eos, length_penalty=alpha)
    assert sorted(eng.free) == free and not eng.tables
    monkeypatch.undo()
    assert eng.beam_search(PROMPTS, beams, steps, eos=eos, length_penalty=alpha) == got     # and with a graph a step
    for logits, scores, cu, out in rec.calls:
        check_select(logits, scores, cu, 2 * beams, out)
    groups = eng_batches(rec.calls)
    want = [h for calls in groups for h in search(calls, beams, eos, alpha, steps)]
    assert [[ids for ids, _ in r] for r in got] == [[h[0] for h in r] for r in want]
    for r, w in zip(got, want):
        for (_, s), (_, t, _) in zip(r, w):
            assert abs(s - t) <= 1e-5 * (1 + abs(t))
    # the logits along a hypothesis, from a pass over its tokens alone
    at = 0
    for calls in groups:
        for b in range(len(calls[0][2]) - 1):
            ids, _, rows = want[at][0]
            s = eng.new()
            for t, (step, row) in enumerate(rows):
                eng.step([(s, PROMPTS[at] if t == 0 else ids[t - 1:t])] if len(PROMPTS[at]) <= 64 or t else
                         [(s, PROMPTS[at][:64])])
                if t == 0 and len(PROMPTS[at]) > 64:
                    eng.step([(s, PROMPTS[at][64:128])])
                    eng.step([(s, PROMPTS[at][128:])])
                a, w = calls[step][0][row].float(), eng.logits[0].float()
                assert ((a - w).norm() / w.norm()).item() < (0.25 if kv == "fp8" else 0.1), (at, t)
            eng.release(s)
            at += 1


def eng_batches(calls):
    """The recorded calls of each batch of prompts: a batch begins with a call of one row a prompt."""
    groups = []
    for c in calls:
        if all(b - a == 1 for a, b in zip(c[2], c[2][1:])) and (not groups or len(groups[-1]) == 12):
            groups.append([])
        groups[-1].append(c)
    return groups


def test_prompts_enter_as_the_pool_allows(monkeypatch):
    """A pool for one prompt's beams at a time gives what a large one gives, but for near-ties of the logits' rounding."""
    few, many = engine(pages=12), engine(pages=300)     # (6, 8 and 6 pages are wanted)
    rec = Record(few, monkeypatch)
    short = [[5, 17, 388, 3], [9] * 40, [400]]
    a = few.beam_search(short, 3, 6)
    assert len([c for c in rec.calls if len(c[2]) == 2]) == 18       # three batches of one
    monkeypatch.undo()
    b = many.beam_search(short, 3, 6)
    for x, y in zip(a, b):
        assert abs(x[0][1] - y[0][1]) < 0.05 * abs(y[0][1])
    assert few.beam_search([], 3, 6) == []


def test_refusals():
    eng = engine(pages=8)
    for bad in (dict(beams=0), dict(beams=33), dict(gen_len=0), dict(length_penalty=-1.0), dict(length_penalty=math.nan), dict(prompts=[[1], []])):
        a = {**dict(prompts=[[1]], beams=2, gen_len=3), **bad}
        with pytest.raises(ValueError):
            eng.beam_search(**a)
    with pytest.raises(RuntimeError, match="pages"):
        eng.beam_search([list(range(100))], 4, 30)
    with pytest.raises(RuntimeError, match="positions"):
        eng.beam_search([[1]], 2, 600)
    assert sorted(eng.free) == list(range(8)) and not eng.tables
