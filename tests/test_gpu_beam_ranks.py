"""The loop's step under torch.distributed (rank 0's candidates for all) takes
the logits that it takes without: any strides."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from graspo_amd import decode_loop as dl

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def test_strided_logits(monkeypatch):
    G, K, V, T = 3, 4, 301, 3
    g = torch.Generator().manual_seed(0)
    prompt = torch.ones(G, 2, dtype=torch.int64, device=DEV)
    xs = [torch.randn(V, G * K, generator=g).to(DEV).t() for _ in range(T)]  # columns apart

    def run(change):
        st = dl.BeamDecodeState(prompt, K, 5, 0, T, 1.0, False)
        got = [st.step(change(x)) for x in xs]
        assert not st.all_done()
        return [(s.tokens, s.parents, *s.state[:5]) for s in got] + [st.finish(2)]

    want = run(torch.Tensor.contiguous)
    alone = run(lambda x: x)
    sent = []
    monkeypatch.setattr(dl, "dist", SimpleNamespace(
        is_available=lambda: True, is_initialized=lambda: True,
        broadcast=lambda t, src: sent.append(src)))
    ranks = [run(lambda x: x), run(lambda x: x.view(G, K, V)), run(torch.Tensor.contiguous)]
    assert sent == [0] * (3 * T * 3)
    for other in (alone, *ranks):
        for a, b in zip(want, other):
            assert all(torch.equal(s, t) for s, t in zip(a, b))
