"""The library's objects go in an order that it can take (plans before their
layer, slabs and layers before their context), whatever order Python finalises
them in: a garbage-collected cycle calls finalisers in any order, and a program
may close its context first.  Runs against a library that records its calls."""
import gc
import itertools

import numpy as np
import pytest

import osm_b200 as osm


class Library:
    def __init__(self):
        self.destroyed, self.names, self.numbers = [], {}, itertools.count(1)

    def __getattr__(self, name):
        def call(*args):
            if name.endswith("_create"):
                args[-1]._obj.value = next(self.numbers)
                self.names[args[-1]._obj.value] = name[4:-7]
            if name.endswith("_destroy"):
                self.destroyed.append(self.names[args[0].value])
            return 0

        return call


@pytest.fixture
def library(monkeypatch):
    gc.collect()
    lib = Library()
    monkeypatch.setattr(osm, "lib", lambda: lib)
    return lib


def make():
    ctx = osm.Context(0, max_tokens=4)
    slab = osm.Slab(ctx, osm.ExpertLayout(), 4)
    layer = osm.Layer(ctx, np.zeros((8, 64), np.float32), 2)
    layer.bind_slab(slab, np.zeros(8, np.int32))
    plan = osm.Plan(layer, 1, None, None)
    return ctx, slab, layer, plan


def in_order(destroyed):
    assert sorted(destroyed) == ["context", "layer", "plan", "slab"]
    at = destroyed.index
    assert at("plan") < at("layer") < at("context") and at("slab") < at("context")


@pytest.mark.parametrize("turn", range(4))
def test_a_collected_cycle(library, turn):
    objects = list(make())
    objects = objects[turn:] + objects[:turn]
    for a, b in zip(objects, objects[1:] + objects[:1]):
        a.other = b
    del a, b, objects
    assert library.destroyed == []
    gc.collect()
    in_order(library.destroyed)


@pytest.mark.parametrize("order", list(itertools.permutations(range(4))))
def test_closed_in_any_order_and_twice(library, order):
    objects = make()
    for i in order:
        objects[i].close()
        objects[i].close()
    in_order(library.destroyed)
    del objects
    gc.collect()
    assert len(library.destroyed) == 4


def test_what_is_not_made_holds_nothing(library, monkeypatch):
    """A slab, layer or plan whose creation fails leaves its context to go."""
    ctx, slab, layer, plan = make()
    for name in ("osm_slab_create", "osm_layer_create", "osm_plan_create"):
        monkeypatch.setattr(library, name, lambda *a: -1, raising=False)
    for f in (lambda: osm.Slab(ctx, osm.ExpertLayout(), 4), lambda: osm.Layer(ctx, np.zeros((8, 64), np.float32), 2),
              lambda: osm.Plan(layer, 1, None, None)):
        with pytest.raises((osm.OsmError, AttributeError)):
            f()
    gc.collect()
    for o in (plan, layer, slab):
        o.close()
    assert library.destroyed == ["plan", "layer", "slab"]
    ctx.close()
    in_order(library.destroyed)
