"""Caches in dicts of every kind keep it.  Without a GPU."""

from collections import OrderedDict, defaultdict

import torch

from graspo_amd.beam_search import map_states


class Named(dict):
    def __init__(self, name):
        super().__init__()
        self.name = name


def test_dicts_of_every_kind():
    t = torch.zeros(2)
    named = Named("layers")
    named["k"] = t
    cache = {"a": defaultdict(list, {3: t, "n": None}), "b": OrderedDict(y=t, x=t + 1), "c": named}
    got = map_states(cache, lambda ts: [v + 10 for v in ts])
    assert type(got["a"]) is defaultdict and got["a"]["missing"] == []
    assert torch.equal(got["a"][3], t + 10) and got["a"]["n"] is None
    assert list(got["b"]) == ["y", "x"] and torch.equal(got["b"]["x"], t + 11)
    assert got["c"].name == "layers" and torch.equal(got["c"]["k"], t + 10)
    # the caller's are as they were
    assert cache["a"][3] is t and cache["c"]["k"] is t and "missing" not in cache["a"]
