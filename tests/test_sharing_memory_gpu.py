"""What the sharing operators' own workspaces hold on to."""
import pytest
import torch

import kernels
from test_paged_gpu import D, DEV, ints, ops
from test_sharing_calls_gpu import check_shared, run_shared
from test_sharing_gpu import check_select, shared_case

pytestmark = pytest.mark.gpu


def test_slowly_growing_calls_keep_one_workspace():
    """Calls of ever more rows: memory for one workspace of the largest call, half as much again at most, and few replacements."""
    k, n_q, V = kernels.DecodeOps(ops().lib), 32, 5000
    pool = torch.randn(40, 8, 16, D, device=DEV).bfloat16()
    q = torch.randn(400, n_q, D, device=DEV).bfloat16()
    out, logits, scores = torch.zeros_like(q), torch.randn(400, V, device=DEV), torch.zeros(400, device=DEV)
    table = torch.arange(40, dtype=torch.int32, device=DEV).view(1, 40)
    sel = torch.zeros(1, 64, device=DEV), *(torch.zeros(1, 64, dtype=torch.int32, device=DEV) for _ in range(2))
    torch.cuda.synchronize()
    before, sizes = torch.cuda.memory_allocated(), set()
    for T in range(20, 401, 20):
        k.shared_attention(q[:T], ints([0, T]), ints([640]), table, ints([0, 1]), ints([0]), pool, pool, out[:T], 0.1, T)
        k.beam_select(logits[:T], scores[:T], ints([0, min(T, 128)]), *sel)
        sizes.add(sum(w.numel() for w in k._scratch.values()))
    most = k.lib.qk_shared_attention_workspace_bytes(400, n_q) + k.lib.qk_beam_workspace_bytes(400, V, 64)
    assert torch.cuda.memory_allocated() - before <= 1.5 * most + (1 << 16) and len(sizes) < 12 and k.device_error() == 0


def test_results_on_a_workspace_that_was_replaced():
    """A small call, a large one that replaces the workspace, a small one on the larger workspace, without a wait between them."""
    k = ops()
    with torch.cuda.stream(torch.cuda.Stream()):
        cases = [shared_case(n, False, way="tensor") for n in ("beams", "large", "drafts")]
        outs = [torch.zeros_like(s["q"]) for s in cases]
        g = torch.Generator(device=DEV).manual_seed(3)
        x = [torch.randn(r, 30000, generator=g, device=DEV) for r in (3, 200, 5)]
        sel = [(torch.zeros(1, 16, device=DEV), *(torch.zeros(1, 16, dtype=torch.int32, device=DEV) for _ in range(2))) for _ in x]
        scores, cu = torch.zeros(200, device=DEV), [ints([0, min(len(y), 128)]) for y in x]
        for i in range(3):
            run_shared(cases[i], outs[i])
            k.beam_select(x[i], scores[:len(x[i])], cu[i], *sel[i])
        torch.cuda.synchronize()
        assert k.device_error() == 0
        for i in range(3):
            check_shared(cases[i], outs[i])
            check_select(x[i], scores[:len(x[i])], cu[i].tolist(), 16, [t.tolist() for t in sel[i]])


def test_calls_take_as_much_of_a_workspace_as_they_need():
    """One buffer, of which each call is given what it needs for its own rows: larger and smaller calls in turn."""
    k = ops()
    cases = [(n, shared_case(n, fp8, seed=i, way=("tensor", "large", "as_it_is")[i % 3]), fp8)
             for i, (n, fp8) in enumerate((n, fp8) for n in ("beams", "large", "mha", "chunks", "drafts") for fp8 in (False, True))]
    size = [k.lib.qk_shared_attention_workspace_bytes(*s["q"].shape[:2]) for _, s, _ in cases]
    assert len(set(size)) > 2
    ws = torch.zeros(max(size), dtype=torch.uint8, device=DEV)
    k.device_error()
    for _ in range(2):
        for n, (name, s, fp8) in zip(size, cases):
            out = torch.zeros_like(s["q"])
            run_shared(s, out, ws[:n])
            assert k.device_error() == 0, name
            check_shared(s, out, fp8)
