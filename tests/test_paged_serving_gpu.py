"""paged.PagedEngine on the GPU: a captured decode step beside passes of other sequences, cuts of a prompt, hand-over to the
contiguous engine (a 2-layer model)."""
import pytest
import torch

import model as M

pytestmark = pytest.mark.gpu


def model():
    return M.Qwen3FP8Decode.synthetic(M.Config(layers=2, vocab=4096), max_seq=512, seed=4, norm_init="random")


def test_the_decode_graph_beside_larger_passes():
    """A graph captured after a short prompt is replayed after passes with more rows: the same tokens and cache as from
    passes alone."""
    from paged import PagedEngine
    short, long = [5, 17, 900, 3], [(13 * i) % 4096 for i in range(200)]
    out = []
    for graph in (True, False):
        eng = PagedEngine(model(), pages=32, page_size=32, max_rows=256)
        s = eng.new()
        toks = eng.step([(s, short)])
        if graph:
            eng.capture([s], toks, 6)
        other = []
        for _ in range(2):
            t = eng.new()
            other += eng.step([(t, long)])
            junk = [torch.full((1 << 20,), 255, dtype=torch.uint8, device="cuda") for _ in range(24)]   # into whatever was freed
            del junk
            if graph:
                toks += eng.decode(3)[0]
            else:
                for _ in range(3):
                    toks += eng.step([(s, toks[-1:])])
        out.append((toks, other, eng.k_pages.clone()))
    assert out[0][:2] == out[1][:2]
    assert torch.equal(out[0][2].view(torch.int16), out[1][2].view(torch.int16))


def test_export_follows_the_contiguous_engine():
    """The exported rows under the reference's own tokens, one by one: its logits at every step."""
    from generate import Engine
    from paged import PagedEngine
    prompt, steps = [(11 * i + 3) % 4096 for i in range(137)], 5
    e = Engine(model())
    e.prefill(prompt, use_graph=False)
    toks, logits = [int(e.token)], []
    for _ in range(steps):
        e.decode_step()
        toks.append(int(e.token))
        logits.append(e.logits.float().clone())
    e.check()
    eng = PagedEngine(model(), pages=16, page_size=32, max_rows=256)
    s = eng.new()
    eng.step([(s, prompt)])
    m = model()
    eng.export(s, m.k_cache[:, 0], m.v_cache[:, 0])
    eng.check()
    e = Engine(m)
    e.state.copy_(torch.tensor([len(prompt), 0], dtype=torch.int32))
    for t, want in zip(toks, logits):
        e.token.fill_(t)
        e.decode_step()
        rel = ((e.logits.float() - want).norm() / want.norm()).item()
        assert rel < 0.1, rel            # W8A8 under other summation orders and fp32 angles
    e.check()


@pytest.mark.parametrize("cut", [1, 50, 136])
def test_a_prompt_in_two_passes(cut):
    """bf16 pages: the logits of a prompt do not depend on where it was cut but for the summation order."""
    from paged import PagedEngine
    prompt = [(17 * i + 5) % 4096 for i in range(137)]
    eng = PagedEngine(model(), pages=16, page_size=32, max_rows=256)
    a, b = eng.new(), eng.new()
    eng.step([(a, prompt)])
    want = eng.logits[0].float().clone()
    eng.step([(b, prompt[:cut])])
    eng.step([(b, prompt[cut:])])
    assert ((eng.logits[0].float() - want).norm() / want.norm()).item() < 0.1
