"""cache_decode with its output on the queries and its weights in place: the
results of the same step into tensors of their own, bit for bit."""
import pytest
import torch

from tests.test_gpu_cache import TYPES, lh, make, step  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("e", TYPES)
def test_out_on_the_queries(lh, e):  # noqa: F811
    for shape in ((3, 2, 8, 128, 70, 200, [0, 100, 200]), (40, 1, 33, 64, 0, 72, [b for b in range(40)]),
                  (2, 1, 71, 96, 129, 131, [131, 5])):
        print(shape[:6], e, flush=True)
        t = make(*shape, TYPES[e], seed=3)
        for weights in (False, True):
            o, w = step(lh, t, weights)
            d = {n: None if x is None else x.cuda() for n, x in t.items()}
            into = d["weights"] if weights else None
            got = lh.cache_decode(d["k"], d["v"], d["q"], d["lens"], d["q"], prefix_k=d["prefix_k"],
                                  prefix_v=d["prefix_v"], weights=into)
            assert got is d["q"] and torch.equal(got, o)
            assert not weights or torch.equal(into, w)


def test_overlaps_are_refused(lh):  # noqa: F811
    t = make(2, 1, 4, 64, 0, 64, [64, 5], torch.bfloat16)
    d = {n: None if x is None else x.cuda() for n, x in t.items()}
    need = lh.cache_decode_workspace_bytes(2, 1, 4, 64, 0, 64)
    ws = torch.zeros(need + 4096, dtype=torch.uint8, device="cuda")
    out = ws[256:256 + 1024].view(torch.bfloat16).view(2, 1, 4, 64)
    with pytest.raises(RuntimeError, match="overlap"):
        lh.cache_decode(d["k"], d["v"], d["q"], d["lens"], out, ws)
    with pytest.raises(RuntimeError, match="overlap"):
        lh.cache_decode(d["k"], d["v"], d["q"], d["lens"], weights=d["weights"], workspace=torch.zeros(
            lh.cache_decode_workspace_bytes(2, 1, 4, 64, 0, 64, True), dtype=torch.uint8, device="cuda"),
                        weights_out=d["v"].view(torch.float32).view(-1)[:128].view(2, 1, 64))
