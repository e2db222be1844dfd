"""The states that follow the beams: whole bytes moved, so every comparison is
exact."""

from __future__ import annotations

import pytest
import torch

from graspo_amd import ops
from graspo_amd.beam_search import expand_states, map_states, reorder_states_

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def values(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    if dtype in (torch.uint8, torch.int32, torch.int64, torch.bool):
        return torch.randint(0, 2 if dtype == torch.bool else 100, shape, generator=g).to(dtype)
    return torch.randn(shape, generator=g).to(dtype)


def maps(G, K, seed):
    """Maps of groups onto themselves: none moves, a step's kind, any, cycles."""
    g = torch.Generator().manual_seed(seed)
    base = torch.arange(G)[:, None] * K
    yield torch.arange(G * K).view(G, K)
    kept = torch.rand(G, K, generator=g) < 0.5
    kept[:, 0] = True
    pick = torch.where(kept, torch.arange(K), kept.float().argmax(1, keepdim=True))
    yield pick + base
    yield torch.randint(0, K, (G, K), generator=g) + base
    yield torch.arange(K).roll(1)[None] + base
    yield torch.arange(K).flip(0)[None] + base


def check(states, G, K, seed=0, parents=None):
    for p in maps(G, K, seed) if parents is None else parents:
        p = p.reshape(-1)
        want = [t.clone()[p.to(DEV)] for t in states]
        reorder_states_(states, p.int().to(DEV), K)
        for t, w in zip(states, want):
            assert torch.equal(t, w)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.uint8, torch.bool,
                                   torch.int64], ids=str)
@pytest.mark.parametrize("G,K", [(1, 1), (1, 2), (3, 4), (2, 8), (2, 16), (2, 17), (1, 33), (1, 64)])
def test_reorder(G, K, dtype):
    print("reorder", G, K, dtype, flush=True)
    shapes = [(3, 5, 8), (1,), (257,), (2, 1000, 16)]
    states = [values((G * K, *s), dtype, i).to(DEV) for i, s in enumerate(shapes)]
    states.append(values((G * K,), dtype, 9).to(DEV))
    check(states, G, K)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.uint8], ids=str)
def test_layouts(dtype):
    G, K = 2, 5
    R = G * K
    guard = 7
    for off in (0, 1, 2, 3):
        for make in (
            lambda b: b[: R * 4 * 40 * 16].view(R, 4, 40, 16)[:, :, :23],       # a filled part
            lambda b: b[: R * 4 * 40 * 16].view(R, 40, 4, 16).transpose(1, 2)[:, :, 3:9],
            lambda b: b[: R * 4 * 40 * 16].view(4, 40, R, 16).permute(2, 0, 1, 3),  # rows inside
            lambda b: b[: R * 4 * 40 * 16].view(40, 16, 4, R).permute(3, 0, 2, 1),  # rows innermost
            lambda b: b[: R * 90].view(R, 90)[:, ::3],
            lambda b: b[: R * 3 * 4 * 5 * 6].view(R, 3, 4, 5, 6)[:, :2, ::2, :3, ::2],
        ):
            buf = torch.full((R * 4 * 40 * 16 + 64,), guard, dtype=dtype, device=DEV)
            t = make(buf[off:])
            t.copy_(values(t.shape, dtype, off))
            outside = torch.ones_like(buf, dtype=torch.bool)
            make(outside[off:]).fill_(False)
            check([t], G, K, seed=off)
            assert buf[outside].eq(guard).all()  # what lies between is left as it was


def test_many_tensors_of_several_shapes():
    G, K = 2, 4
    states = []
    for i in range(230):  # more than one launch holds
        states.append(values((8, 2, 3 + i % 3 // 2, 8), torch.bfloat16, i).to(DEV))
    check(states, G, K)


def test_a_state_past_32_bit_offsets():
    G, K = 1, 3
    t = torch.zeros(3, (1 << 31) + 64, dtype=torch.uint8, device=DEV)
    t[:, -64:] = values((3, 64), torch.uint8, 1).to(DEV)
    t[:, :64] = values((3, 64), torch.uint8, 2).to(DEV)
    p = torch.tensor([2, 0, 1])
    want = t[:, -64:].clone()[p.to(DEV)], t[:, :64].clone()[p.to(DEV)]
    reorder_states_([t], p.int().to(DEV), K)
    assert torch.equal(t[:, -64:], want[0]) and torch.equal(t[:, :64], want[1])


def test_parents_outside_their_group():
    t = torch.arange(6, device=DEV).view(6, 1).float()
    for bad in ([0, 1, 2, 3, 4, 2], [-1, 1, 2, 3, 4, 5], [0, 1, 6, 3, 4, 5], [0, 1, 2, 3, 1 << 30, 5]):
        for dt in (torch.int32, torch.int64):
            s = t.clone()
            with pytest.raises(RuntimeError, match="outside its row's group"):
                reorder_states_([s], torch.tensor(bad, dtype=dt, device=DEV), 3)
            assert torch.equal(s, t)
    s = t.clone()
    reorder_states_([s], torch.tensor([1, 1, 9, 4, 3, 3], dtype=torch.int32, device=DEV), 3,
                    check_status=False)
    assert s.flatten().tolist() == [1, 1, 2, 4, 3, 3]
    with pytest.raises(RuntimeError, match="outside"):
        reorder_states_([s], torch.tensor([2 ** 33, 1], dtype=torch.int64, device=DEV).repeat(3), 2)


def test_refusals():
    t = torch.zeros(4, 8, device=DEV)
    p = torch.arange(4, dtype=torch.int32, device=DEV)
    for states in ([t, t], [t, t[:, 4:]], [t[:1].expand(4, 8)], [t.as_strided((4, 8), (4, 1))]):
        with pytest.raises(RuntimeError, match="overlap"):
            reorder_states_(states, p, 2)
    reorder_states_([t[:, :4], t[:, 4:]], p, 2)  # columns of one buffer
    with pytest.raises(RuntimeError, match="rows"):
        reorder_states_([t, torch.zeros(3, 8, device=DEV)], p, 2)
    with pytest.raises(RuntimeError, match="rows"):
        reorder_states_([torch.zeros((), device=DEV)], p, 2)
    with pytest.raises(RuntimeError, match="beams"):
        reorder_states_([torch.zeros(65, 2, device=DEV)], torch.arange(65, device=DEV), 65)
    with pytest.raises(RuntimeError, match="gradient"):
        reorder_states_([torch.zeros(4, 8, device=DEV, requires_grad=True)], p, 2)
    for bad in (p.float(), p.view(2, 2)):
        with pytest.raises(ValueError, match="parents"):
            reorder_states_([t], bad, 2)
    with pytest.raises(ValueError, match="groups"):
        reorder_states_([t], p, 3)


def test_nothing_to_move():
    reorder_states_([], torch.zeros(0, dtype=torch.int32, device=DEV), 4)
    p = torch.zeros(0, dtype=torch.int32, device=DEV)
    reorder_states_([torch.zeros(0, 8, device=DEV)], p, 4)
    reorder_states_([torch.zeros(4, 0, device=DEV)], torch.arange(4, device=DEV).int(), 4)
    assert expand_states([], 3) == []
    assert expand_states([torch.zeros(0, 5, device=DEV)], 3)[0].shape == (0, 5)
    assert expand_states([torch.zeros(2, 0, device=DEV)], 3)[0].shape == (6, 0)


def test_written_in_place_is_seen():
    t = torch.randn(4, 8, device=DEV, requires_grad=True)
    c = t * 1.0
    out = (c * c).sum()  # saves c
    with torch.no_grad():
        reorder_states_([c.detach()], torch.tensor([0, 0, 2, 2], device=DEV), 2)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.backward()
    with torch.inference_mode():
        s = torch.arange(4.0, device=DEV).view(4, 1)
        reorder_states_([s], torch.tensor([1, 1, 3, 2], device=DEV), 2)
        assert s.flatten().tolist() == [1, 1, 3, 2]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.uint8, torch.int64], ids=str)
@pytest.mark.parametrize("G,K", [(1, 1), (1, 4), (3, 5), (2, 64)])
def test_expand(G, K, dtype):
    for make in (lambda b: b.view(G, 4, 30, 16), lambda b: b.view(G, 4, 30, 16)[:, :, 1:18],
                 lambda b: b.view(G, 30, 4, 16).transpose(1, 2), lambda b: b.view(G, -1)[:, 3:47:2],
                 lambda b: b.view(30, 16, 4, G).permute(3, 2, 0, 1), lambda b: b.view(G, -1)[:, 5],
                 lambda b: b.view(G, -1)[:, :1].expand(G, 7)):
        t = make(values((G * 4 * 30 * 16,), dtype, 1).to(DEV))
        u = make(values((G * 4 * 30 * 16,), dtype, 2).to(DEV))
        for got, want in zip(expand_states([t, u], K), (t, u)):
            assert got.is_contiguous() and torch.equal(got, want.repeat_interleave(K, 0))


def test_captured_and_replayed():
    G, K = 2, 4
    t = values((8, 3, 64), torch.bfloat16, 0).to(DEV)
    p = torch.arange(8, dtype=torch.int32, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        reorder_states_([t], p, K)  # (does not wait in a capture)
        out = expand_states([t], 2)
    for i, m in enumerate(maps(G, K, 3)):
        new = values((8, 3, 64), torch.bfloat16, i).to(DEV)
        t.copy_(new)
        p.copy_(m.reshape(-1))
        graph.replay()
        torch.cuda.synchronize()
        want = new[m.reshape(-1).to(DEV)]
        assert torch.equal(t, want) and torch.equal(out[0], want.repeat_interleave(2, 0))


def test_nested_caches():
    a, b = torch.zeros(2, 3), torch.ones(2)
    cache = [(a, None), {"k": b, "n": 4}]
    got = map_states(cache, lambda ts: [t + 1 for t in ts])
    assert torch.equal(got[0][0], a + 1) and got[0][1] is None
    assert torch.equal(got[1]["k"], b + 1) and got[1]["n"] == 4
    with pytest.raises(TypeError, match="cache"):
        map_states([object()], lambda ts: ts)


def test_copies_have_storages_of_their_own():
    states = [values((2, 5, 7), dt, 0).to(DEV) for dt in (torch.float32, torch.bfloat16, torch.uint8)]
    outs = expand_states(states, 3)
    assert len({t.untyped_storage().data_ptr() for t in outs}) == 3
    for t in outs:
        assert t.storage_offset() == 0
        assert t.untyped_storage().nbytes() == t.numel() * t.element_size()
