"""beam_select where masks are large finite numbers in place of -inf: tokens, whole rows and beams at the type's lowest value. Bounds as
in test_sharing_gpu.py; the 64-bit scores take a row's maximum off first, as a sum beside the lowest value is lost in 64 bits too."""
import math

import pytest
import torch

from test_paged_gpu import DEV
from test_sharing_gpu import select

pytestmark = pytest.mark.gpu


def check_masked(logits, scores, cu, k, got):
    """As check_select, for scores of any size."""
    x = logits.double()
    y = x - x.amax(1, keepdim=True)
    lp = scores.double()[:, None] + (y - y.exp().sum(1, keepdim=True).log())
    lp = lp.masked_fill(lp.float() == -math.inf, -math.inf)          # (out of the outputs' range)
    V = logits.shape[1]
    for b, (lo, hi) in enumerate(zip(cu, cu[1:])):
        s, parent, token = (g[b] for g in got)
        best = lp[lo:hi].flatten().topk(min(k, (hi - lo) * V)).values.tolist()
        best = [v for v in best if v > -math.inf]
        assert [p >= 0 for p in parent] == [i < len(best) for i in range(k)], b
        assert len(set(zip(parent, token))) >= len(best)
        for i, want in enumerate(best):
            e = lp[parent[i], token[i]].item()
            tol = abs(e) * 2.0 ** -24 + 2.0 ** -17
            assert abs(s[i] - e) <= tol and abs(e - want) <= 2 * tol, (b, i, s[i], e, want)
        for r in range(lo, hi):
            mine = [t for p, t in zip(parent, token) if p == r]
            assert mine == torch.sort(x[r], descending=True, stable=True).indices[:len(mine)].tolist(), (b, r, mine)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("V,rows", [(100, 4), (5000, 3), (40000, 20)])
@pytest.mark.parametrize("kind", ["a_row", "a_row_that_is_best", "tokens", "all_rows", "-1e30", "-1e9_row"])
def test_select_masked_by_large_numbers(kind, V, rows, dtype):
    g = torch.Generator(device=DEV).manual_seed(V + rows)
    low = {"-1e30": -1e30, "-1e9_row": -1e9}.get(kind, torch.finfo(dtype).min)
    logits, scores, k = (torch.randn(rows, V, generator=g, device=DEV) * 3).to(dtype), torch.randn(rows, generator=g, device=DEV) - 15, 24
    if kind in ("a_row", "-1e30", "-1e9_row"):
        logits[1] = low
    elif kind == "a_row_that_is_best":
        logits[1] = low
        scores[1] = -2.0
    elif kind == "all_rows":
        logits.fill_(low)
    else:
        logits[:, 5:] = low                         # five tokens a row are left
    if kind == "-1e9_row":
        logits[1, V // 2:] += 1e8                   # a row that lies low as a whole still has an order
    err, got = select(logits, scores, [0, 2, rows], k)
    assert err == 0
    check_masked(logits, scores, [0, 2, rows], k, got)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_select_beams_of_a_low_score(dtype):
    """Beams that a caller keeps out by a score of -1e9: they come behind all others, and only where those are too few."""
    g = torch.Generator(device=DEV).manual_seed(6)
    logits = torch.randn(8, 12, generator=g, device=DEV).to(dtype)
    scores = torch.tensor([0.0, -1e9, -1e9, -1e9] * 2, device=DEV)
    err, got = select(logits, scores, [0, 4, 8], 20)
    assert err == 0 and all(p[:12] == [r] * 12 for p, r in zip(got[1], (0, 4)))
    check_masked(logits, scores, [0, 4, 8], 20, got)


@pytest.mark.parametrize("V", [300, 50000])
@pytest.mark.parametrize("score", [-1e12, -3e38, -15.0])
def test_select_scores_that_swallow_the_logits(score, V):
    """Equal scores in 64 bits, because a beam's score so far or the other logits are far larger: a row keeps the order of its logits."""
    g = torch.Generator(device=DEV).manual_seed(V)
    logits = torch.rand(3, V, generator=g, device=DEV) * (1e-7 if score < -100 else 1e-18)
    scores = torch.full((3,), score, device=DEV)
    err, got = select(logits, scores, [0, 3], 40)
    assert err == 0
    check_masked(logits, scores, [0, 3], 40, got)
