"""What Context.q4_gemv_lora, Context.route_scores, Lora and Routing check before
the library is called, case by case, without a GPU: the arguments are CPU
tensors that say they are on the GPU, and the library is one that records its
calls, so every refusal is the named check's and every accepted call gets
through."""
import pytest
import torch

import osm_b200 as osm


class OnGpu:
    """A CPU tensor that reports CUDA device `index`."""

    def __init__(self, t, index=0):
        self.t, self.index = t, index
        self.is_cuda, self.device = True, torch.device("cuda", index)

    def get_device(self):
        return self.index

    def __getitem__(self, i):
        return OnGpu(self.t[i], self.index)

    def __getattr__(self, name):
        return getattr(self.t, name)


class Library:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return 0

        return call


@pytest.fixture
def library(monkeypatch):
    lib = Library()
    monkeypatch.setattr(osm, "lib", lambda: lib)
    return lib


@pytest.fixture
def ctx(library):
    c = object.__new__(osm.Context)
    c.h, c.device, c.max_tokens = None, 0, 4
    return c


def projection(**change):
    """Arguments of a projection of 4 tokens, 128 to 32, with three adapters."""
    v = dict(packed=OnGpu(torch.zeros(32, 16, dtype=torch.int32)),
             scales=OnGpu(torch.zeros(32, 2, dtype=torch.bfloat16)),
             biases=OnGpu(torch.zeros(32, 2, dtype=torch.bfloat16)), out_dim=32, in_dim=128,
             x=OnGpu(torch.zeros(4, 128)), tokens=4, y=OnGpu(torch.zeros(4, 32)),
             lora=osm.Lora(OnGpu(torch.zeros(3, 8, 128, dtype=torch.bfloat16)),
                           OnGpu(torch.zeros(3, 32, 8, dtype=torch.bfloat16))),
             adapter=OnGpu(torch.zeros(4, dtype=torch.int32)))
    v.update(change)
    return v


def project(ctx, v):
    ctx.q4_gemv_lora(v["packed"], v["scales"], v["biases"], v["out_dim"], v["in_dim"], v["x"], v["tokens"], v["y"],
                     lora=v["lora"], adapter=v["adapter"])


def test_projection_is_called(ctx, library):
    v = projection()
    project(ctx, v)
    (name, args), = library.calls
    assert name == "osm_q4_gemv_lora"
    assert args[1:4] == tuple(v[k].data_ptr() for k in ("packed", "scales", "biases"))
    assert args[4:11] == (32, 128, 64, v["x"].data_ptr(), 0, 128, 4) and args[13:] == (v["y"].data_ptr(), 32)


@pytest.mark.parametrize("packed,scales", [(torch.int32, torch.bfloat16), (torch.uint32, torch.uint16),
                                           (torch.uint8, torch.uint8), (torch.int32, torch.int16)])
def test_q4_tables_in_the_types_that_hold_them(ctx, library, packed, scales):
    """Words, or the bytes of a slot; bf16, or its bits."""
    n = 4 if packed == torch.uint8 else 1
    m = 2 if scales == torch.uint8 else 1
    tables = dict(packed=OnGpu(torch.zeros(32 * 16 * n, dtype=packed)),
                  scales=OnGpu(torch.zeros(32 * 2 * m, dtype=scales)),
                  biases=OnGpu(torch.zeros(32 * 2 * m + 5, dtype=scales)))
    project(ctx, projection(**tables))
    assert len(library.calls) == 1


@pytest.mark.parametrize("name,table", [
    ("packed", OnGpu(torch.zeros(31, 16, dtype=torch.int32))), ("packed", OnGpu(torch.zeros(32, 16))),
    ("packed", OnGpu(torch.zeros(32 * 16 * 4 - 1, dtype=torch.uint8))),
    ("packed", OnGpu(torch.zeros(32, 32, dtype=torch.int32)[:, ::2])), ("packed", torch.zeros(32, 16, dtype=torch.int32)),
    ("packed", OnGpu(torch.zeros(32, 16, dtype=torch.int32), index=1)),
    ("scales", OnGpu(torch.zeros(32, 1, dtype=torch.bfloat16))), ("scales", OnGpu(torch.zeros(32, 2))),
    ("scales", OnGpu(torch.zeros(32, 2, dtype=torch.float16))), ("scales", torch.zeros(32, 2, dtype=torch.bfloat16)),
    ("biases", OnGpu(torch.zeros(63, dtype=torch.uint16))),
    ("biases", OnGpu(torch.zeros(32, 4, dtype=torch.bfloat16)[:, ::2])),
    ("biases", OnGpu(torch.zeros(32, 2, dtype=torch.bfloat16), index=1))])
def test_q4_tables_that_do_not_hold_the_weights(ctx, library, name, table):
    """Short, of another type, strided, on the CPU or on another device."""
    with pytest.raises(ValueError, match=name):
        project(ctx, projection(**{name: table}))
    assert not library.calls


def route(ctx, tokens=None, routing=None, **change):
    """64 experts, top 8, 4 tokens."""
    v = dict(logits=OnGpu(torch.zeros(4, 64)), ids=OnGpu(torch.zeros(4, 8, dtype=torch.int32)),
             weights=OnGpu(torch.zeros(4, 8)), mass=OnGpu(torch.zeros(4)))
    v.update(change)
    ctx.route_scores(v["logits"], routing or osm.Routing(64, 8), v["ids"], v["weights"], mass=v["mass"], tokens=tokens)


def test_routing_is_called(ctx, library):
    route(ctx)
    route(ctx, tokens=3, logits=OnGpu(torch.zeros(4, 70)[:, :64]))
    assert [(n, a[3:6]) for n, a in library.calls] == [("osm_route_scores", (0, 64, 4)), ("osm_route_scores", (0, 70, 3))]


@pytest.mark.parametrize("tokens", [-1, -2**31, -2**32 + 4, 5])
def test_token_counts(ctx, library, tokens):
    """Counts that are more than the rows, and negative ones, which the
    library's unsigned count would take as billions of rows."""
    with pytest.raises(ValueError, match="rows|token"):
        route(ctx, tokens=tokens)
    with pytest.raises(ValueError, match="rows|token"):
        project(ctx, projection(tokens=tokens))
    assert not library.calls


@pytest.mark.parametrize("field", ["experts", "top_k", "groups", "top_groups"])
@pytest.mark.parametrize("value", [-1, 2**32 + 1])
def test_routing_fields_that_would_wrap(field, value):
    """2**32 + 1 groups are not one group."""
    with pytest.raises(ValueError, match=field):
        osm.Routing(**{**dict(experts=64, top_k=8, groups=2, top_groups=1), field: value})


# ---- each check of test_serving_refusals by its own reason ----

A, B = (3, 8, 128), (3, 32, 8)


def table(a_type=torch.bfloat16, b_type=torch.bfloat16, a=None, b=None, **kw):
    a = torch.zeros(A, dtype=a_type) if a is None else a
    b = torch.zeros(B, dtype=b_type) if b is None else b
    return osm.Lora(OnGpu(a), OnGpu(b), **kw)


def half(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


def test_adapter_table_is_accepted():
    t = table(scale=OnGpu(torch.ones(3)), ranks=OnGpu(torch.ones(3, dtype=torch.int32)))
    assert (t.desc.count, t.desc.rank, t.desc.a_stride, t.desc.b_stride) == (3, 8, 8 * 128, 32 * 8)
    t = table(a=half(3, 9, 128)[:, :8], b=half(3, 40, 8)[:, :32])   # gaps between adapters
    assert (t.desc.a_stride, t.desc.b_stride) == (9 * 128, 40 * 8)


@pytest.mark.parametrize("reason,kwargs", [
    ("bf16 or fp16", dict(a_type=torch.float32, b_type=torch.float32)),
    ("A and B alike", dict(b_type=torch.float16)),
    (r"B \[n\]\[out\]\[rank\]", dict(b=half(3, 32, 7))), (r"B \[n\]\[out\]\[rank\]", dict(b=half(2, 32, 8))),
    ("must be contiguous", dict(a=half(3, 128, 8).transpose(1, 2))),
    ("must be contiguous", dict(b=half(3, 32, 16)[:, :, ::2])),
    ("must not overlap", dict(a=half(1, 8, 128).expand(A))), ("must not overlap", dict(b=half(1, 32, 8).expand(B))),
    ("adapter scale", dict(scale=OnGpu(torch.ones(2)))), ("adapter scale", dict(scale=OnGpu(torch.ones(3).double()))),
    ("adapter scale: not on", dict(scale=OnGpu(torch.ones(3), index=1))),
    ("adapter ranks", dict(ranks=OnGpu(torch.ones(3)))), ("adapter ranks: not on", dict(ranks=torch.ones(3, dtype=torch.int32)))])
def test_adapter_table_refused_for(reason, kwargs):
    with pytest.raises(ValueError, match=reason):
        table(**kwargs)


def test_adapters_of_two_devices_or_none():
    for a, b in ((half(*A), half(*B)), (OnGpu(half(*A)), OnGpu(half(*B), index=1))):
        with pytest.raises(ValueError, match="on one GPU"):
            osm.Lora(a, b)


@pytest.mark.parametrize("x,expected", [(torch.zeros(4, 64), (0, 64)), (torch.zeros(4, 70)[:, :64].bfloat16(), (1, 64)),
                                        (torch.zeros(4, 70, dtype=torch.float16)[:, :64], (2, 70)),
                                        (torch.zeros(9, 64)[::2], (0, 128))])
def test_rows_are_accepted(x, expected):
    assert osm._rows(OnGpu(x), 64, 4, 0, "x") == expected


@pytest.mark.parametrize("reason,x", [
    ("fp32, bf16 or fp16", OnGpu(torch.zeros(4, 64, dtype=torch.int32))),
    ("4 rows of 64", OnGpu(torch.zeros(4, 60))), ("4 rows of 64", OnGpu(torch.zeros(3, 64))),
    ("4 rows of 64", OnGpu(torch.zeros(256))), ("must be contiguous", OnGpu(torch.zeros(64, 4).t())),
    ("must not overlap", OnGpu(torch.zeros(1, 64).expand(4, 64))), ("not on the context's device", torch.zeros(4, 64)),
    ("not on the context's device", OnGpu(torch.zeros(4, 64), index=1))])
def test_rows_refused_for(reason, x):
    with pytest.raises(ValueError, match=reason):
        osm._rows(x, 64, 4, 0, "x")


@pytest.mark.parametrize("reason,change", [
    ("ids", dict(ids=OnGpu(torch.zeros(4, 7, dtype=torch.int32)))), ("ids", dict(ids=OnGpu(torch.zeros(4, 8, dtype=torch.int64)))),
    ("weights", dict(weights=OnGpu(torch.zeros(4, 16)[:, ::2]))), ("weights", dict(weights=torch.zeros(4, 8))),
    ("mass", dict(mass=OnGpu(torch.zeros(3)))), ("logits", dict(logits=OnGpu(torch.zeros(4, 63))))])
def test_routing_arguments_refused_for(ctx, library, reason, change):
    with pytest.raises(ValueError, match=f"route.* {reason}"):
        route(ctx, **change)
    assert not library.calls


@pytest.mark.parametrize("reason,change", [
    ("of one type", dict(y=OnGpu(torch.zeros(4, 32).bfloat16()))), ("another projection", dict(out_dim=31, y=OnGpu(torch.zeros(4, 31)))),
    ("indices are missing", dict(adapter=None)), ("adapter", dict(adapter=OnGpu(torch.zeros(4, dtype=torch.int64)))),
    ("adapter", dict(adapter=OnGpu(torch.zeros(3, dtype=torch.int32)))), ("x: 4 rows", dict(x=OnGpu(torch.zeros(3, 128)))),
    ("y: 4 rows", dict(y=OnGpu(torch.zeros(4, 33))))])
def test_projection_arguments_refused_for(ctx, library, reason, change):
    with pytest.raises(ValueError, match=reason):
        project(ctx, projection(**change))
    assert not library.calls


def test_routing_choices_and_bias(ctx, library):
    for kw in (dict(score="tanh"), dict(group_score="mean")):
        with pytest.raises(ValueError, match="score is softmax or sigmoid"):
            osm.Routing(64, 8, **kw)
    for bias in (OnGpu(torch.zeros(63)), OnGpu(torch.zeros(64).half()), torch.zeros(64)):
        with pytest.raises(ValueError, match="routing bias"):
            osm.Routing(64, 8, bias=bias)
    route(ctx, routing=osm.Routing(64, 8, bias=OnGpu(torch.zeros(64))))
    with pytest.raises(ValueError, match="bias: not on the context's device"):
        route(ctx, routing=osm.Routing(64, 8, bias=OnGpu(torch.zeros(64), index=1)))
    assert len(library.calls) == 1
