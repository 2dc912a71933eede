"""beam_select over several chunks of a row in one CTA: candidates that come late, few at a time or many at once. Bounds as in
test_sharing_gpu.py."""
import pytest
import torch

from test_paged_gpu import DEV, cumulative, ints, ops
from test_sharing_gpu import check_select

pytestmark = pytest.mark.gpu


def select_again(logits, scores, cu, k, times):
    """Calls on one workspace; the results of the first, which the others have to give to the bit."""
    o, B = ops(), len(cu) - 1
    ws = o.beam_workspace(DEV, *logits.shape, k)
    outs = [(torch.full((B, k), 7.0, device=DEV), *(torch.full((B, k), 7, dtype=torch.int32, device=DEV) for _ in range(2))) for _ in range(times)]
    o.device_error()
    for out in outs:
        o.beam_select(logits, scores, ints(cu), *out, workspace=ws)
    assert o.device_error() == 0
    assert all(torch.equal(a, b) for out in outs for a, b in zip(out, outs[0]))
    return tuple(t.tolist() for t in outs[0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("rows,some,k", [(300, 0.06, 16), (300, 0.01, 64), (180, 0.09, 8), (700, 0.04, 33)])
def test_dense_chunks_behind_sparse_ones(rows, some, k, dtype):
    """Every CTA has 5 chunks of a row or more: in each a share of the 16-byte vectors is above all before it, and in one chunk of a
    row, somewhere, all are. So the vectors kept aside are few at one look at them and too many at the next."""
    V, size = 151936, 16 // dtype.itemsize
    chunk = V // -(-V // (2048 * size))             # (about)
    g = torch.Generator(device=DEV).manual_seed(rows + k)
    logits = (torch.randn(rows, V, generator=g, device=DEV) * 0.1).to(dtype)
    at = torch.arange(V, device=DEV) // chunk
    vectors = torch.rand(rows, V // size, generator=g, device=DEV) < some
    lift = vectors.repeat_interleave(size, 1) & (torch.arange(V, device=DEV) % size == 3)
    logits += (lift * (2 + at * 0.25)).to(dtype)
    dense = torch.randint(2, int(at[-1]) + 1, (rows, 1), generator=g, device=DEV)
    logits += ((at == dense) * (2 + at * 0.25)).to(dtype)
    scores = torch.randn(rows, generator=g, device=DEV) * 0.5 - 9
    cu = cumulative([min(60, rows - i) for i in range(0, rows, 60)])
    check_select(logits, scores, cu, k, select_again(logits, scores, cu, k, 20))


def test_the_most_chunks_of_a_call():
    """65,536 rows of 1,048,576 fp32 values (one row, at a stride of 0): 8,454,144 chunks, whose products with the CTAs pass 2^31."""
    rows, V, k = 65536, 1 << 20, 2
    g = torch.Generator(device=DEV).manual_seed(7)
    row = torch.randn(1, V, generator=g, device=DEV)
    scores = torch.randn(rows, generator=g, device=DEV)
    cu = list(range(0, rows + 1, 128))
    out = select_again(row.expand(rows, V), scores, cu, k, 1)
    best = row[0].topk(2)
    lp = best.values.double() - torch.logsumexp(row[0].double(), 0)
    s = scores.view(-1, 128).double()
    for b, (at, want) in enumerate(zip(s.argmax(1).tolist(), (s.amax(1) + lp[0]).tolist())):
        assert (out[1][b][0], out[2][b][0]) == (cu[b] + at, best.indices[0].item()), b
        assert abs(out[0][b][0] - want) <= abs(want) * 2.0 ** -24 + 2.0 ** -17
