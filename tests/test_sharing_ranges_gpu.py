"""shared_attention where one CTA's or warp's range of work holds pieces of different kinds: groups of different sizes behind each
other, units cut between CTAs. Bounds as in test_sharing_gpu.py."""
import pytest
import torch

import test_sharing_gpu
from test_paged_gpu import D, DEV, attend64, check_attention, ints, ops
from test_sharing_calls_gpu import check_shared, run_shared
from test_sharing_gpu import shared_case

pytestmark = pytest.mark.gpu

# as SHARED in test_sharing_gpu.py. A tile pair of the tensor cores holds a prefix's rows in one tile, twice or four times where they are few
# (up to 16 tokens at 4 heads a KV head), once from there on, and in both tiles from 33 tokens on.
CHANGES = {
    "long": ([(22, 8192), (14, 8192), (20, 8192)], [1], [30, 5], 32, 8, 64),
    "both_tiles": ([(22, 4096), (40, 4096), (7, 4096), (70, 4096), (12, 4096), (33, 4096)], [1], [30, 5], 32, 8, 16),
    "short": ([(n, 256 + 128 * (i % 2)) for i in range(17) for n in (18, 5, 17, 36, 20, 9)], [1], [1, 7], 16, 4, 128),
    "short_mha": ([(n, 256) for _ in range(4) for n in (70, 20, 100, 40, 130)], [1], [3], 4, 4, 32),
    "drafts": ([(6, 2048), (2, 2048), (9, 1024), (3, 4096), (5, 2048)], [4, 1, 3, 5], [40, 6], 32, 8, 32),
}


@pytest.mark.parametrize("way", ["as_it_is", "tensor"])
@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("name", CHANGES)
def test_groups_of_different_sizes_in_one_range(name, fp8, way, monkeypatch):
    monkeypatch.setitem(test_sharing_gpu.SHARED, name, CHANGES[name])
    k = ops()
    s = shared_case(name, fp8, way=way)
    ws = k.shared_workspace(DEV, *s["q"].shape[:2])
    outs = [torch.full_like(s["q"], 3.0) for _ in range(5)]
    k.device_error()
    for out in outs:
        run_shared(s, out, ws)
    assert k.device_error() == 0
    assert (outs[0][s["cu"][-1]:] == 3).all() and all(torch.equal(out, outs[0]) for out in outs)
    check_shared(s, outs[0], fp8)


# Chunks of prompts behind a shared one: sequences with more than 64 query rows a KV head are the tensor cores' for their own keys too, and
# with 1,000 own keys and more (8 key tiles) they are cut between CTAs, beside sequences that are not cut, and some in no group.
CHUNKS = {
    "one_long": ([(2, 1024)], [1024, 1], [1500, 9], 32, 8, 64),
    "several": ([(3, 512), (2, 1280), (2, None)], [300, 40, 1, 513, 128], [2000, 45, 1100, 1030, 900], 32, 8, 16),
    "few_rows_of_long_own": ([(4, 2048)], [17, 33, 20, 65], [4000, 1025, 2050, 1200], 32, 8, 128),
    "mha": ([(3, 640)], [200, 70, 129], [1300, 1100, 129], 4, 4, 32),
    "one_kv_head": ([(5, 1024), (2, 256)], [64, 3, 90, 5, 400], [3000, 50, 1024, 1700, 400], 16, 1, 64),
    "group_5": ([(3, 768)], [150, 14, 13], [1500, 1300, 40], 10, 2, 32),
}


@pytest.mark.parametrize("way", ["as_it_is", "large", "tensor"])
@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("name", CHUNKS)
def test_long_chunks_behind_a_shared_prefix(name, fp8, way, monkeypatch):
    monkeypatch.setitem(test_sharing_gpu.SHARED, name, CHUNKS[name])
    k = ops()
    s = shared_case(name, fp8, way=way)
    ws = k.shared_workspace(DEV, *s["q"].shape[:2])
    outs = [torch.full_like(s["q"], 3.0) for _ in range(3)]
    k.device_error()
    for out in outs:
        run_shared(s, out, ws)
    assert k.device_error() == 0
    assert (outs[0][s["cu"][-1]:] == 3).all() and all(torch.equal(out, outs[0]) for out in outs)
    check_shared(s, outs[0], fp8)


@pytest.mark.parametrize("max_q", [3, 200])
@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "e4m3"])
def test_rows_that_see_nothing(fp8, max_q, monkeypatch):
    """Sequences shorter than their new tokens, or empty: the first rows give zeros, as in paged_attention, beside a shared prefix."""
    monkeypatch.setitem(test_sharing_gpu.SHARED, "short", ([(30, 1280), (5, None)], [1, max_q], [200], 32, 8, 32))
    k = ops()
    s = shared_case("short", fp8)
    n, lens = s["n"], s["lens"]
    for b, length in ((30, 0), (31, max_q - 2), (33, 1), (34, 0)):
        lens[b] = length
        s["rows"][b] = [x[:length] for x in s["rows"][b]]
    out, want = torch.full_like(s["q"], 3.0), torch.full_like(s["q"], 3.0)
    k.device_error()
    run_shared(s, out)
    k.paged_attention(s["q"], ints(s["cu"]), ints(lens), s["table"], s["k"], s["v"], want, D ** -0.5, max_q, k_scale=s["ks"], v_scale=s["vs"])
    assert k.device_error() == 0
    for b, length in ((30, 0), (31, max_q - 2), (33, 1), (34, 0)):
        a, z = s["cu"][b], s["cu"][b + 1]
        hidden = z - a - length                     # rows of the sequence that see nothing
        assert (out[a:a + hidden] == 0).all() and (want[a:a + hidden] == 0).all() and (out[a + hidden:z] != 0).any(-1).all()
    keep = [b for b in range(30)] + [32]
    check_attention(torch.cat([out[s["cu"][b]:s["cu"][b + 1]] for b in keep]), *(torch.cat(x) for x in zip(*[
        attend64(s["q"][s["cu"][b]:s["cu"][b + 1]].double(), *s["rows"][b], lens[b] - n[b], D ** -0.5) for b in keep])), fp8)
