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
