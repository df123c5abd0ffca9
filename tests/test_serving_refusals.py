"""Refusals of osm_route_scores, osm_moe_route_scores and osm_q4_gemv_lora that
need no GPU: missing contexts, and tables that the Python classes turn down."""
import ctypes

import pytest
import torch

import osm_b200 as osm
from osm_b200 import _lib, build


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def test_no_context(lib):
    routing, table = _lib.RoutingDesc(), _lib.LoraDesc()
    buf = ctypes.addressof(ctypes.create_string_buffer(64))
    assert lib.osm_route_scores(None, ctypes.byref(routing), buf, 0, 0, 1, buf, buf, None) == lib.osm_route_scores(
        None, None, None, 0, 0, 0, None, None, None) != 0
    assert lib.osm_moe_route_scores(None, ctypes.byref(routing), buf, 1, buf, buf, None) != 0
    assert lib.osm_q4_gemv_lora(None, buf, buf, buf, 64, 64, 64, buf, 0, 0, 1, ctypes.byref(table), buf, buf, 0) != 0


@pytest.mark.parametrize("kwargs", [dict(score="tanh"), dict(group_score="mean"), dict(bias=torch.zeros(8)),
                                    dict(bias=torch.zeros(8, dtype=torch.float16))])
def test_routing(kwargs):
    with pytest.raises(ValueError):
        osm.Routing(8, 2, **kwargs)


def test_routing_fields():
    r = osm.Routing(64, 6, score="sigmoid", groups=8, top_groups=3, group_score="top2", renormalize=False, scale=2.5)
    d = r.desc
    assert (d.experts, d.top_k, d.groups, d.top_groups, d.renormalize, d.scale) == (64, 6, 8, 3, 0, 2.5)
    assert d.score == _lib.OSM_SCORE_SIGMOID and d.group_score == _lib.OSM_GROUP_TOP2 and not d.balance_bias_dev
    assert osm.Routing(64, 6, groups=4).desc.top_groups == 4


@pytest.mark.parametrize("change", ["float", "types", "shape", "inner", "overlap", "cpu"])
def test_adapter_tables(change):
    a = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    b = torch.zeros(3, 32, 4, dtype=torch.bfloat16)
    if change == "float":
        a, b = a.float(), b.float()
    if change == "types":
        b = b.half()
    if change == "shape":
        b = b[:, :, :3]
    if change == "inner":
        a = a.transpose(1, 2).contiguous().transpose(1, 2)
    if change == "overlap":
        a = a[:1].expand(3, 4, 64)
    with pytest.raises(ValueError):
        osm.Lora(a, b)


@pytest.mark.parametrize("x", [torch.zeros(4, 64, dtype=torch.int32), torch.zeros(4, 60), torch.zeros(3, 64),
                               torch.zeros(64, 4).t(), torch.zeros(1, 64).expand(4, 64), torch.zeros(256),
                               torch.zeros(4, 64)])
def test_rows(x):
    """Rows of another type, length, count, order, that overlap, flat, or not on the GPU."""
    with pytest.raises(ValueError):
        osm._rows(x, 64, 4, 0, "x")
